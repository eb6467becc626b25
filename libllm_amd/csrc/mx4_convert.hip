// Matrices into MXFP4 and back (mx4.h says what that is and how it lies).
//
// Quantising: s = floor(log2(max |x|)) - 2 over a block, at least -127, so that the largest
// magnitude falls into 4 .. 8, of which 6 is the largest code; then every element divided by 2^s,
// rounded to the nearest code, ties to the even one, what lies beyond 6 to 6.  The exponent comes
// from the bits of the largest magnitude and the division by a power of two is exact, so there is
// one rounding, the format's own.  A block that holds an infinity or a NaN has no such scale: it is
// marked 255 and reads as NaN.
//
// One pass over memory each way, which bounds both.  A block takes a tile of 16 rows by a quad of units
// (512 elements of K), a wave a unit, so that codes move 1 KiB in a row and scales as one word a lane.  Where
// rows allow it a lane takes 16 bytes of a row and its neighbours the rest of the line (reading back by a lane's
// whole block, 64 lines apart an instruction, held that kernel to 1.8 TB/s): quantising, four neighbouring lanes share a
// block, find its largest magnitude between them, and their codes meet through shared memory.  Rows that do
// not begin at multiples of 8 bytes go element by element, neighbours in neighbouring lanes, through shared
// memory.  28,672 x 4,096 in bfloat16: 62 us to codes and 54 back (4.8 and 5.5 TB/s; a plain copy 5.1), in
// float32 108 and 98; 8 x 2,048: 3.0 and 2.3, a launch.
#include "mx4.h"

#define CV_LD 132           // floats a row of a unit takes in shared memory: 128, and 4 that shift the banks

// Unit u of rows row0 .. row0 + 15, element by element into shared memory (zero where there are none).
template <typename T>
__device__ __forceinline__ void stage_rows(const T* X, size_t ldx, int M, int K, int row0, int u, int lane, float* mine) {
  const int k = u * MX4_UNIT + lane;
  const int ka = min(k, K - 1), kb = min(k + 64, K - 1);       // (no load hangs on a condition: all of them go out at once)
  T a[16], b[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const T* p = X + (size_t)min(row0 + i, M - 1) * ldx;
    a[i] = p[ka];
    b[i] = p[kb];
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const bool on = row0 + i < M;
    mine[i * CV_LD + lane] = on && k < K ? Conv<T>::load(&a[i]) : 0.f;
    mine[i * CV_LD + lane + 64] = on && k + 64 < K ? Conv<T>::load(&b[i]) : 0.f;
  }
}

// The scale byte of a block from the bits of its largest magnitude.
__device__ __forceinline__ uint32_t block_scale(uint32_t top) {
  const uint32_t e = top >> 23;
  return e == 255 ? 255u : (e > 2 ? e - 2 : 0u);
}

__device__ __forceinline__ uint32_t code8(const float* v, float scale) {
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], scale, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], scale, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], scale, 3);
}

// Eight neighbours, BYTES at a time (8 or 16).  In bfloat16 sixteen lanes read whole lines, which nobody reads
// again here: past the caches (28,672 x 4,096: 62 us against 71).
template <int BYTES> __device__ __forceinline__ void load8(const float* p, float* v) {
#pragma unroll
  for (int j = 0; j < 8; j += 4) {
    const float4 q = Conv4<float>::load(p + j);
    v[j] = q.x; v[j + 1] = q.y; v[j + 2] = q.z; v[j + 3] = q.w;
  }
}
template <int BYTES> __device__ __forceinline__ void load8(const bf16_t* p, float* v) {
  uint32_t w[4];
  if constexpr (BYTES == 16) {
    const u32x4_raw q = __builtin_nontemporal_load(reinterpret_cast<const u32x4_raw*>(p));
    w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
  } else {
    const uint2 a = *reinterpret_cast<const uint2*>(p), b = *reinterpret_cast<const uint2*>(p + 4);
    w[0] = a.x; w[1] = a.y; w[2] = b.x; w[3] = b.y;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = __uint_as_float(w[j] << 16);
    v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
  }
}

#define CV_CODES (3 * 80 + 64)          // words of a unit's codes in shared memory, the four blocks of a row in different banks

// BYTES: what rows are aligned to, 16 or 8, or 0 for neither.
template <typename T, int BYTES>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const T* __restrict__ X, size_t ldx, int M, int K,
                                                           uint4* __restrict__ codes, uint32_t* __restrict__ scales,
                                                           int quads) {
  __shared__ __attribute__((aligned(16))) float lds[BYTES ? 4 * CV_CODES : 4 * 16 * CV_LD];
  __shared__ uint32_t s_scale[64];                            // byte i of word l: wave i's scale of its lane l
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int tile = blockIdx.x, quad = blockIdx.y, u = quad * 4 + wave;
  uint8_t* scale_of = reinterpret_cast<uint8_t*>(s_scale) + wave;
  uint4 mine;
  // (a wave's accesses to shared memory run in order; the compiler may not move a lane's read over another's write)
  if constexpr (BYTES != 0) {
    uint32_t* words = reinterpret_cast<uint32_t*>(lds) + wave * CV_CODES;
    const int g = (lane >> 2) & 3, j = lane & 3, k = u * MX4_UNIT + (lane & 15) * 8;
    float v[4][8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = tile * 16 + i * 4 + (lane >> 4);
      const T* p = X + (size_t)row * ldx + k;
      if (row < M && k + 8 <= K) {
        load8<BYTES>(p, v[i]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = row < M && k + e < K ? Conv<T>::load(p + e) : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i * 4 + (lane >> 4);
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[i][e]) & 0x7fffffffu);
      top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xf, 0xf, false));    // lane ^ 1
      top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xf, 0xf, false));    // lane ^ 2
      const uint32_t scale = block_scale(top);
      words[g * 80 + r * 4 + j] = code8(v[i], mx4_scale(scale));
      if (j == 0) scale_of[(g * 16 + r) * 4] = (uint8_t)scale;
    }
    asm volatile("" ::: "memory");
    mine = *reinterpret_cast<const uint4*>(words + (lane >> 4) * 80 + (lane & 15) * 4);
  } else {
    float* rows = lds + wave * 16 * CV_LD;
    stage_rows<T>(X, ldx, M, K, tile * 16, u, lane, rows);
    asm volatile("" ::: "memory");
    float v[MX4_BLOCK];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < MX4_BLOCK; j += 4) {
      const float4 q = *reinterpret_cast<const float4*>(rows + (lane & 15) * CV_LD + (lane >> 4) * MX4_BLOCK + j);
      v[j] = q.x; v[j + 1] = q.y; v[j + 2] = q.z; v[j + 3] = q.w;
    }
#pragma unroll
    for (int j = 0; j < MX4_BLOCK; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
    const uint32_t scale = block_scale(top);
    const float sf = mx4_scale(scale);
    mine = make_uint4(code8(v, sf), code8(v + 8, sf), code8(v + 16, sf), code8(v + 24, sf));
    scale_of[lane * 4] = (uint8_t)scale;
  }
  codes[((size_t)tile * quads * 4 + u) * 64 + lane] = mine;
  __syncthreads();
  if (wave == 0) scales[((size_t)tile * quads + quad) * 64 + lane] = s_scale[lane];
}

// WIDE: a lane makes 16 bytes of a row, else 8 elements through shared memory.  PAST: they are written past
// the caches, which would not hold them for the reader (us alone, and with a copy of the result after it: 28,672
// x 4,096 in bfloat16, 235 MB, 54 / 153 against 73 / 169; 12,288 x 8,192, 201 MB, the copy too 130 against 142; but
// 8,192 x 8,192, 134 MB, 83 against 79).
template <typename T, bool WIDE, bool PAST>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(const uint32_t* __restrict__ codes,
                                                             const uint32_t* __restrict__ scales, T* __restrict__ out,
                                                             int M, int K, int quads) {
  __shared__ __attribute__((aligned(16))) float lds[WIDE ? 4 : 4 * 16 * CV_LD];
  constexpr int PER = WIDE && sizeof(T) == 4 ? 4 : 8;         // neighbouring elements a lane
  constexpr int LPR = MX4_UNIT / PER, RPP = 64 / LPR, PASSES = 16 / RPP;      // lanes a row, rows a pass
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int tile = blockIdx.x, quad = blockIdx.y, u = quad * 4 + wave;
  const int piece = lane % LPR, word = piece * PER / 8, g = word >> 2, j = word & 3;
  const int k = u * MX4_UNIT + piece * PER;
  if (u * MX4_UNIT >= K) return;
  float* mine = lds + (WIDE ? 0 : wave * 16 * CV_LD);
  uint32_t sw[PASSES], w[PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int at = g * 16 + i * RPP + lane / LPR;
    sw[i] = scales[((size_t)tile * quads + quad) * 64 + at];
    w[i] = codes[(((size_t)tile * quads * 4 + u) * 64 + at) * 4 + j];
    if (PER == 4) w[i] >>= 16 * (lane & 1);
  }
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int r = i * RPP + lane / LPR, row = tile * 16 + r;
    const float sf = mx4_scale((sw[i] >> (8 * wave)) & 255u);
    const f32x2_raw a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], sf, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], sf, 1);
    const f32x2_raw c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], sf, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], sf, 3);
    if constexpr (!WIDE) {
      *reinterpret_cast<float4*>(mine + r * CV_LD + piece * 8) = make_float4(a.x, a.y, b.x, b.y);
      *reinterpret_cast<float4*>(mine + r * CV_LD + piece * 8 + 4) = make_float4(c.x, c.y, d.x, d.y);
    } else if (row < M && k < K) {                            // K is a multiple of PER here
      u32x4_raw q;
      if constexpr (PER == 8) q = u32x4_raw{pack2_bf16(a.x, a.y), pack2_bf16(b.x, b.y), pack2_bf16(c.x, c.y), pack2_bf16(d.x, d.y)};
      else q = u32x4_raw{__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y)};
      u32x4_raw* dst = reinterpret_cast<u32x4_raw*>(out + (size_t)row * K + k);
      if constexpr (PAST) __builtin_nontemporal_store(q, dst);
      else *dst = q;
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
// file holds them, into the tiles.  Once for a weight: sixteen loads of a byte a lane, whatever rows are aligned to
// (28,672 x 4,096: 107 us, 1.2 TB/s).
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
  // (two neighbours a thread and store, eight loads at once; ldo is even)
  for (size_t m = blockIdx.x; m < (size_t)M; m += gridDim.x) {
    const bf16_t* x = X + m * ldx;
    for (int k0 = (blockIdx.y * 1024 + threadIdx.x) * 2; k0 < ldo; k0 += gridDim.y * 2048) {
      uint32_t lo[4], hi[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        lo[i] = x[min(k0 + i * 512, K - 1)];
        hi[i] = x[min(k0 + i * 512 + 1, K - 1)];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = k0 + i * 512;
        if (k < ldo) *reinterpret_cast<uint32_t*>(out + m * ldo + k) = (k < K ? lo[i] : 0) | (k + 1 < K ? hi[i] << 16 : 0);
      }
    }
  }
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
  const size_t at = (uintptr_t)X | ldx * (dtype == LLM_DTYPE_F32 ? 4 : 2);
#define MX4_LAUNCH(T, BYTES) \
  mx4_quantize_kernel<T, BYTES><<<grid, 256, 0, stream>>>((const T*)X, ldx, M, K, (uint4*)codes, (uint32_t*)scales, quads)
  if (dtype == LLM_DTYPE_F32) {
    if (at % 16 == 0) MX4_LAUNCH(float, 16); else MX4_LAUNCH(float, 0);
  } else if (dtype == LLM_DTYPE_BF16) {
    if (at % 16 == 0) MX4_LAUNCH(bf16_t, 16); else if (at % 8 == 0) MX4_LAUNCH(bf16_t, 8); else MX4_LAUNCH(bf16_t, 0);
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
  const bool past = (size_t)M * K * (dtype == LLM_DTYPE_F32 ? 4 : 2) >= (size_t)192 << 20;      // three quarters of the last-level cache
#define MX4_LAUNCH(T, W, P) \
  mx4_dequantize_kernel<T, W, P><<<grid, 256, 0, stream>>>((const uint32_t*)codes, (const uint32_t*)scales, (T*)out, M, K, quads)
#define MX4_LAUNCH_T(T) \
  do { if (!wide) MX4_LAUNCH(T, false, false); else if (past) MX4_LAUNCH(T, true, true); else MX4_LAUNCH(T, true, false); } while (0)
  if (dtype == LLM_DTYPE_F32) MX4_LAUNCH_T(float);
  else if (dtype == LLM_DTYPE_BF16) MX4_LAUNCH_T(bf16_t);
  else return LLM_ERR_ARG;
#undef MX4_LAUNCH_T
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
  if (K <= 0 || ldx < (size_t)K || ldo < K || (ldo & 1) || X == nullptr || out == nullptr || (((uintptr_t)out) & 3)) return LLM_ERR_ARG;
  const dim3 grid(M < (1 << 16) ? M : 1 << 16, ldo < (1 << 19) ? (ldo + 2047) / 2048 : 256);
  pad_rows_kernel<<<grid, 256, 0, stream>>>((const bf16_t*)X, ldx, (bf16_t*)out, M, K, ldo);
  return llm_launch_status();
}
