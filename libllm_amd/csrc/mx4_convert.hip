// Matrices into MXFP4 and back (mx4.h says what that is and how it lies).
//
// Quantising: s = floor(log2(max |x|)) - 2 over a block, at least -127, so that the largest
// magnitude falls into 4 .. 8, of which 6 is the largest code; then every element divided by 2^s,
// rounded to the nearest code, ties to the even one, what lies beyond 6 to 6.  The exponent comes
// from the bits of the largest magnitude and the division by a power of two is exact, so there is
// one rounding, the format's own.  A block that holds an infinity or a NaN has no such scale: it is
// marked 255 and reads as NaN.
//
// One pass over memory each way.  A block takes a tile of 16 rows by a quad of units (512 elements of
// K), a wave a unit, so that codes move 1 KiB in a row and scales as one word a lane.  Quantising, lane l has block
// l / 16 of row l % 16 of each unit, as the tiles lie; reading back, a lane makes 8 neighbouring
// elements, 16 lanes a row of 128, so that a store takes whole lines (stores of a lane's whole block,
// 64 lines apart an instruction, held the kernel to 1.8 TB/s).  Rows that do not begin at multiples of
// 16 bytes go element by element, neighbours in neighbouring lanes, through shared memory.
// 28,672 x 4,096 in bfloat16: 69 us to codes and 68 back (4.3 and 4.4 TB/s of 5.1 for a plain copy);
// 8 x 2,048: 3.0 and 2.3, a launch.
#include "mx4.h"

#define CV_LD 132           // floats a row of a unit takes in shared memory: 128, and 4 that shift the banks

// Unit u of rows row0 .. row0 + 15, element by element into shared memory (zero where there are none).
template <typename T>
__device__ __forceinline__ void stage_rows(const T* X, size_t ldx, int M, int K, int row0, int u, int lane, float* mine) {
  const int k = u * MX4_UNIT + lane;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const bool on = row0 + i < M;
    const T* p = X + (size_t)(row0 + i) * ldx + k;
    const float a = on && k < K ? Conv<T>::load(p) : 0.f, b = on && k + 64 < K ? Conv<T>::load(p + 64) : 0.f;
    mine[i * CV_LD + lane] = a;
    mine[i * CV_LD + lane + 64] = b;
  }
}

template <typename T, bool WIDE>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const T* __restrict__ X, size_t ldx, int M, int K,
                                                           uint4* __restrict__ codes, uint32_t* __restrict__ scales,
                                                           int quads) {
  __shared__ __attribute__((aligned(16))) float lds[WIDE ? 4 : 4 * 16 * CV_LD];
  __shared__ uint32_t s_scale[64];                            // byte i of word l: wave i's scale of its lane l
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int tile = blockIdx.x, quad = blockIdx.y, r = lane & 15, g = lane >> 4;
  float* mine = lds + (WIDE ? 0 : wave * 16 * CV_LD);
  const int row = tile * 16 + r, u = quad * 4 + wave;
  const int k = u * MX4_UNIT + g * MX4_BLOCK;
  const int n = row < M ? K - k : 0;
  const T* p = X + (size_t)row * ldx + k;
  float v[MX4_BLOCK];
  if (!WIDE) {
    // (a wave's accesses to shared memory run in order; the compiler may not move a lane's read over another's write)
    stage_rows<T>(X, ldx, M, K, tile * 16, u, lane, mine);
    asm volatile("" ::: "memory");
  }
  if (!WIDE || n >= MX4_BLOCK) {
#pragma unroll
    for (int j = 0; j < MX4_BLOCK; j += 4) {
      const float4 q = WIDE ? Conv4<T>::load(p + j) : *reinterpret_cast<const float4*>(mine + r * CV_LD + g * MX4_BLOCK + j);
      v[j] = q.x; v[j + 1] = q.y; v[j + 2] = q.z; v[j + 3] = q.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < MX4_BLOCK; ++j) v[j] = j < n ? Conv<T>::load(p + j) : 0.f;
  }
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < MX4_BLOCK; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
  const uint32_t e = top >> 23;
  const uint32_t scale = e == 255 ? 255u : (e > 2 ? e - 2 : 0u);
  const float sf = mx4_scale(scale);
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[8 * j], v[8 * j + 1], sf, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[8 * j + 2], v[8 * j + 3], sf, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[8 * j + 4], v[8 * j + 5], sf, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[8 * j + 6], v[8 * j + 7], sf, 3);
    w[j] = c;
  }
  codes[((size_t)tile * quads * 4 + u) * 64 + lane] = make_uint4(w[0], w[1], w[2], w[3]);
  reinterpret_cast<uint8_t*>(s_scale)[lane * 4 + wave] = (uint8_t)scale;
  __syncthreads();
  if (wave == 0) scales[((size_t)tile * quads + quad) * 64 + lane] = s_scale[lane];
}

template <typename T, bool WIDE>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(const uint32_t* __restrict__ codes,
                                                             const uint32_t* __restrict__ scales, T* __restrict__ out,
                                                             int M, int K, int quads) {
  __shared__ __attribute__((aligned(16))) float lds[WIDE ? 4 : 4 * 16 * CV_LD];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int tile = blockIdx.x, quad = blockIdx.y, u = quad * 4 + wave;
  const int piece = lane & 15, g = piece >> 2, j = piece & 3;         // this lane's 8 elements of a row's 128
  const int k = u * MX4_UNIT + piece * 8;
  if (u * MX4_UNIT >= K) return;
  float* mine = lds + (WIDE ? 0 : wave * 16 * CV_LD);
  uint32_t sw[4], w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = g * 16 + i * 4 + (lane >> 4);
    sw[i] = scales[((size_t)tile * quads + quad) * 64 + at];
    w[i] = codes[(((size_t)tile * quads * 4 + u) * 64 + at) * 4 + j];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = i * 4 + (lane >> 4), row = tile * 16 + r;
    const float sf = mx4_scale((sw[i] >> (8 * wave)) & 255u);
    const f32x2_raw a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], sf, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], sf, 1);
    const f32x2_raw c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], sf, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], sf, 3);
    if (!WIDE) {
      *reinterpret_cast<float4*>(mine + r * CV_LD + piece * 8) = make_float4(a.x, a.y, b.x, b.y);
      *reinterpret_cast<float4*>(mine + r * CV_LD + piece * 8 + 4) = make_float4(c.x, c.y, d.x, d.y);
      continue;
    }
    if (row >= M || k >= K) continue;
    T* dst = out + (size_t)row * K + k;
    if (sizeof(T) == 2) {                                     // K is a multiple of 8 here
      *reinterpret_cast<uint4*>(dst) = make_uint4(pack2_bf16(a.x, a.y), pack2_bf16(b.x, b.y), pack2_bf16(c.x, c.y), pack2_bf16(d.x, d.y));
    } else {                                                  // and here of 4
      Conv4<T>::store(dst, make_float4(a.x, a.y, b.x, b.y));
      if (k + 4 < K) Conv4<T>::store(dst + 4, make_float4(c.x, c.y, d.x, d.y));
    }
  }
  if (!WIDE) {
    asm volatile("" ::: "memory");
    const int at = u * MX4_UNIT + lane;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int row = tile * 16 + i;
      const float a = mine[i * CV_LD + lane], b = mine[i * CV_LD + lane + 64];
      if (row < M && at < K) Conv<T>::store(out + (size_t)row * K + at, a);
      if (row < M && at + 64 < K) Conv<T>::store(out + (size_t)row * K + at + 64, b);
    }
  }
}

// Codes [N, ldc] bytes (two elements a byte, the even one low) and scales [N, ceil(K / 32)] as a
// file holds them, into the tiles.
__global__ __launch_bounds__(256) void mx4_pack_kernel(const uint8_t* __restrict__ rows, size_t ldc,
                                                       const uint8_t* __restrict__ row_scales, int N, int K,
                                                       uint4* __restrict__ codes, uint32_t* __restrict__ scales,
                                                       int quads) {
  __shared__ uint32_t s_scale[64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int tile = blockIdx.x, quad = blockIdx.y, r = lane & 15, g = lane >> 4;
  const int row = tile * 16 + r, blocks = (K + MX4_BLOCK - 1) / MX4_BLOCK;
  const int u = quad * 4 + wave, b = u * 4 + g;
  uint32_t w[4] = {0, 0, 0, 0};
  uint8_t scale = 0;
  if (row < N && b < blocks) {
    const uint8_t* src = rows + (size_t)row * ldc + b * 16;
    const int left = K - b * MX4_BLOCK;                         // elements of the row from this block on
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      uint32_t byte = 2 * j < left ? src[j] : 0u;
      if (2 * j + 1 >= left) byte &= 15u;
      w[j >> 2] |= byte << (8 * (j & 3));
    }
    scale = row_scales[(size_t)row * blocks + b];
  }
  codes[((size_t)tile * quads * 4 + u) * 64 + lane] = make_uint4(w[0], w[1], w[2], w[3]);
  reinterpret_cast<uint8_t*>(s_scale)[lane * 4 + wave] = scale;
  __syncthreads();
  if (wave == 0) scales[((size_t)tile * quads + quad) * 64 + lane] = s_scale[lane];
}

// Rows of K bfloat16 elements into rows of K rounded up to 8, the elements added zero: for the
// products, which read 16 bytes at a time, where K or the address is no multiple of that.
__global__ __launch_bounds__(256) void pad_rows_kernel(const bf16_t* __restrict__ X, size_t ldx,
                                                       bf16_t* __restrict__ out, int M, int K, int ldo) {
  for (size_t m = blockIdx.x; m < (size_t)M; m += gridDim.x)
    for (int k = blockIdx.y * 256 + threadIdx.x; k < ldo; k += gridDim.y * 256)
      out[m * ldo + k] = k < K ? X[m * ldx + k] : (bf16_t)0;
}

static inline dim3 mx4_grid(int rows, int k) { return dim3(mx4_tiles(rows), mx4_quads(k)); }

// X [M, K] of `dtype`, rows ldx elements apart, into codes (mx4_tiles(M) * mx4_quads(K) * 4096 bytes)
// and scales (mx4_tiles(M) * mx4_quads(K) * 256 bytes).
extern "C" int llm_mx4_quantize(const void* X, int dtype, size_t ldx, int M, int K, void* codes, void* scales,
                                hipStream_t stream) {
  if (M <= 0 || K <= 0 || ldx < (size_t)K || X == nullptr || codes == nullptr || scales == nullptr) return LLM_ERR_ARG;
  if ((((uintptr_t)codes) | ((uintptr_t)scales)) & 15) return LLM_ERR_ARG;
  const dim3 grid = mx4_grid(M, K);
  if (grid.y > 65535) return LLM_ERR_ARG;
  const int quads = mx4_quads(K);
  const bool wide = (ldx & 3) == 0 && (((uintptr_t)X) & (dtype == LLM_DTYPE_F32 ? 15 : 7)) == 0;
#define MX4_LAUNCH(T, W) \
  mx4_quantize_kernel<T, W><<<grid, 256, 0, stream>>>((const T*)X, ldx, M, K, (uint4*)codes, (uint32_t*)scales, quads)
  if (dtype == LLM_DTYPE_F32) {
    if (wide) MX4_LAUNCH(float, true); else MX4_LAUNCH(float, false);
  } else if (dtype == LLM_DTYPE_BF16) {
    if (wide) MX4_LAUNCH(bf16_t, true); else MX4_LAUNCH(bf16_t, false);
  } else {
    return LLM_ERR_ARG;
  }
#undef MX4_LAUNCH
  return llm_launch_status();
}

extern "C" int llm_mx4_dequantize(const void* codes, const void* scales, void* out, int dtype, int M, int K,
                                  hipStream_t stream) {
  if (M <= 0 || K <= 0 || out == nullptr || codes == nullptr || scales == nullptr) return LLM_ERR_ARG;
  if ((((uintptr_t)codes) | ((uintptr_t)scales)) & 15) return LLM_ERR_ARG;
  const dim3 grid = mx4_grid(M, K);
  if (grid.y > 65535) return LLM_ERR_ARG;
  const int quads = mx4_quads(K);
  const bool wide = (K & (dtype == LLM_DTYPE_F32 ? 3 : 7)) == 0 && (((uintptr_t)out) & 15) == 0;
#define MX4_LAUNCH(T, W) \
  mx4_dequantize_kernel<T, W><<<grid, 256, 0, stream>>>((const uint32_t*)codes, (const uint32_t*)scales, (T*)out, M, K, quads)
  if (dtype == LLM_DTYPE_F32) {
    if (wide) MX4_LAUNCH(float, true); else MX4_LAUNCH(float, false);
  } else if (dtype == LLM_DTYPE_BF16) {
    if (wide) MX4_LAUNCH(bf16_t, true); else MX4_LAUNCH(bf16_t, false);
  } else {
    return LLM_ERR_ARG;
  }
#undef MX4_LAUNCH
  return llm_launch_status();
}

extern "C" int llm_mx4_pack(const void* rows, size_t ldc, const void* row_scales, int N, int K, void* codes,
                            void* scales, hipStream_t stream) {
  if (N <= 0 || K <= 0 || ldc < (size_t)((K + 1) / 2) || rows == nullptr || row_scales == nullptr || codes == nullptr ||
      scales == nullptr)
    return LLM_ERR_ARG;
  if ((((uintptr_t)codes) | ((uintptr_t)scales)) & 15) return LLM_ERR_ARG;
  const dim3 grid = mx4_grid(N, K);
  if (grid.y > 65535) return LLM_ERR_ARG;
  mx4_pack_kernel<<<grid, 256, 0, stream>>>((const uint8_t*)rows, ldc, (const uint8_t*)row_scales, N, K, (uint4*)codes,
                                            (uint32_t*)scales, mx4_quads(K));
  return llm_launch_status();
}

extern "C" int llm_pad_rows(const void* X, size_t ldx, void* out, int M, int K, int ldo, hipStream_t stream) {
  if (M <= 0) return LLM_OK;
  if (K <= 0 || ldx < (size_t)K || ldo < K || X == nullptr || out == nullptr) return LLM_ERR_ARG;
  const dim3 grid(M < (1 << 16) ? M : 1 << 16, ldo < (1 << 19) ? (ldo + 2047) / 2048 : 256);
  pad_rows_kernel<<<grid, 256, 0, stream>>>((const bf16_t*)X, ldx, (bf16_t*)out, M, K, ldo);
  return llm_launch_status();
}
