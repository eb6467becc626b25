// Matrices into MXFP4 and back (mx4.h says what that is and how it lies).
//
// Quantising: s = floor(log2(max |x|)) - 2 over a block, at least -127, so that the largest
// magnitude falls into 4 .. 8, of which 6 is the largest code; then every element divided by 2^s,
// rounded to the nearest code, ties to the even one, what lies beyond 6 to 6.  The exponent comes
// from the bits of the largest magnitude and the division by a power of two is exact, so there is
// one rounding, the format's own.  A block that holds an infinity or a NaN has no such scale: it is
// marked 255 and reads as NaN.
//
// All three kernels are one pass over memory.  A wave takes a tile of 16 rows by four units (512
// elements of K): lane l has block l / 16 of row l % 16 of each unit, as the tiles lie, so that the
// codes go out in stores of 1 KiB in a row and the scales as one word a lane.
#include "mx4.h"

// 32 elements of a row from `p`, of which the first `n` exist (the rest are zero), as floats.
template <typename T, bool WIDE>
__device__ __forceinline__ void block_load(const T* p, int n, float (&v)[MX4_BLOCK]) {
  if (WIDE && n >= MX4_BLOCK) {
#pragma unroll
    for (int i = 0; i < MX4_BLOCK; i += 4) {
      const float4 q = Conv4<T>::load(p + i);
      v[i] = q.x; v[i + 1] = q.y; v[i + 2] = q.z; v[i + 3] = q.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < MX4_BLOCK; ++i) v[i] = i < n ? Conv<T>::load(p + i) : 0.f;
  }
}

template <typename T, bool WIDE>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const T* __restrict__ X, size_t ldx, int M, int K,
                                                           uint4* __restrict__ codes, uint32_t* __restrict__ scales,
                                                           int quads) {
  const int lane = threadIdx.x & 63, quad = blockIdx.y * 4 + (threadIdx.x >> 6);
  const int tile = blockIdx.x, r = lane & 15, g = lane >> 4;
  if (quad >= quads) return;
  const int row = tile * 16 + r;
  uint32_t sw = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int u = quad * 4 + i;
    const int k = u * MX4_UNIT + g * MX4_BLOCK;
    const int n = row < M ? K - k : 0;
    float v[MX4_BLOCK];
    block_load<T, WIDE>(X + (size_t)row * ldx + k, n, v);
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
    sw |= scale << (8 * i);
  }
  scales[((size_t)tile * quads + quad) * 64 + lane] = sw;
}

template <typename T, bool WIDE>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(const uint4* __restrict__ codes,
                                                             const uint32_t* __restrict__ scales, T* __restrict__ out,
                                                             int M, int K, int quads) {
  const int lane = threadIdx.x & 63, quad = blockIdx.y * 4 + (threadIdx.x >> 6);
  const int tile = blockIdx.x, r = lane & 15, g = lane >> 4;
  const int row = tile * 16 + r;
  if (quad >= quads || row >= M) return;
  const uint32_t sw = scales[((size_t)tile * quads + quad) * 64 + lane];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int u = quad * 4 + i;
    const int k = u * MX4_UNIT + g * MX4_BLOCK, n = K - k;
    if (n <= 0) break;
    const uint4 c = codes[((size_t)tile * quads * 4 + u) * 64 + lane];
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
    const float sf = mx4_scale((sw >> (8 * i)) & 255u);
    float v[MX4_BLOCK];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f32x2_raw p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[j], sf, 0);
      v[8 * j] = p.x; v[8 * j + 1] = p.y;
      p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[j], sf, 1);
      v[8 * j + 2] = p.x; v[8 * j + 3] = p.y;
      p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[j], sf, 2);
      v[8 * j + 4] = p.x; v[8 * j + 5] = p.y;
      p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[j], sf, 3);
      v[8 * j + 6] = p.x; v[8 * j + 7] = p.y;
    }
    T* dst = out + (size_t)row * K + k;
    if (WIDE && n >= MX4_BLOCK) {
#pragma unroll
      for (int j = 0; j < MX4_BLOCK; j += 4) Conv4<T>::store(dst + j, make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]));
    } else {
#pragma unroll
      for (int j = 0; j < MX4_BLOCK; ++j)
        if (j < n) Conv<T>::store(dst + j, v[j]);
    }
  }
}

// Codes [N, ldc] bytes (two elements a byte, the even one low) and scales [N, ceil(K / 32)] as a
// file holds them, into the tiles.
__global__ __launch_bounds__(256) void mx4_pack_kernel(const uint8_t* __restrict__ rows, size_t ldc,
                                                       const uint8_t* __restrict__ row_scales, int N, int K,
                                                       uint4* __restrict__ codes, uint32_t* __restrict__ scales,
                                                       int quads) {
  const int lane = threadIdx.x & 63, quad = blockIdx.y * 4 + (threadIdx.x >> 6);
  const int tile = blockIdx.x, r = lane & 15, g = lane >> 4;
  if (quad >= quads) return;
  const int row = tile * 16 + r, blocks = (K + MX4_BLOCK - 1) / MX4_BLOCK;
  uint32_t sw = 0;
  for (int i = 0; i < 4; ++i) {
    const int u = quad * 4 + i, b = u * 4 + g;
    uint32_t w[4] = {0, 0, 0, 0};
    if (row < N && b < blocks) {
      const uint8_t* src = rows + (size_t)row * ldc + b * 16;
      const int left = K - b * MX4_BLOCK;                       // elements of the row from this block on
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        uint32_t byte = 2 * j < left ? src[j] : 0u;
        if (2 * j + 1 >= left) byte &= 15u;
        w[j >> 2] |= byte << (8 * (j & 3));
      }
      sw |= (uint32_t)row_scales[(size_t)row * blocks + b] << (8 * i);
    }
    codes[((size_t)tile * quads * 4 + u) * 64 + lane] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  scales[((size_t)tile * quads + quad) * 64 + lane] = sw;
}

// Rows of K bfloat16 elements into rows of K rounded up to 8, the elements added zero: for the
// products, which read 16 bytes at a time, where K or the address is no multiple of that.
__global__ __launch_bounds__(256) void pad_rows_kernel(const bf16_t* __restrict__ X, size_t ldx,
                                                       bf16_t* __restrict__ out, int K, int ldo) {
  const size_t m = blockIdx.x;
  for (int k = blockIdx.y * 256 + threadIdx.x; k < ldo; k += gridDim.y * 256)
    out[m * ldo + k] = k < K ? X[m * ldx + k] : (bf16_t)0;
}

static inline dim3 mx4_grid(int rows, int k) { return dim3(mx4_tiles(rows), (mx4_quads(k) + 3) / 4); }

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
  const bool wide = (K & 3) == 0 && (((uintptr_t)out) & 15) == 0;
#define MX4_LAUNCH(T, W) \
  mx4_dequantize_kernel<T, W><<<grid, 256, 0, stream>>>((const uint4*)codes, (const uint32_t*)scales, (T*)out, M, K, quads)
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
  pad_rows_kernel<<<dim3(M, (ldo + 2047) / 2048), 256, 0, stream>>>((const bf16_t*)X, ldx, (bf16_t*)out, K, ldo);
  return llm_launch_status();
}
