// Matrices in microscaled 4-bit floating point (MXFP4): what a code stands for, and how they lie.
//
// Every 32 neighbouring elements of a row (a block; the last of a row may be shorter) share a scale
// 2^(e - 127), e a byte (255: the block reads as NaN), and an element is four bits: a sign and one
// of the magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6.
//
// A matrix [R, K] is kept in tiles of 16 rows by units of 128 elements of K, as the matrix cores
// take it: per (tile, unit) 64 pieces of 16 bytes, piece l holding the block l / 16 of row l % 16,
// element j of the block in bits 4 (j % 8) .. + 3 of word j / 8.  That is the operand of lane l for
// v_mfma_scale_f32_16x16x128_f8f6f4, and word j of every piece is the operand of one
// v_mfma_f32_16x16x32_bf16 once it is widened (its slots of K then stand for the elements
// 32 (l / 16) + 8 j .. + 7 of the unit, for which the other operand is read the same way).  A wave's
// load of a unit is 1 KiB in a row.  The scales of four units in a row (a quad) lie together, a word
// a lane: byte u % 4 of word ((tile * quads + u / 4) * 64 + lane).  A tile has whole quads; rows,
// blocks and elements that pad it are zero.
#pragma once
#include "mfma.h"

#define MX4_BLOCK 32
#define MX4_UNIT 128
__host__ __device__ inline int mx4_tiles(int rows) { return (rows + 15) / 16; }
__host__ __device__ inline int mx4_units(int k) { return (k + MX4_UNIT - 1) / MX4_UNIT; }
__host__ __device__ inline int mx4_quads(int k) { return (mx4_units(k) + 3) / 4; }

typedef int i32x8_raw __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_raw __attribute__((ext_vector_type(2)));
typedef float f32x2_raw __attribute__((ext_vector_type(2)));

// The scale byte as the float that the conversions below take: they use its exponent alone, so 0
// is 2^-127 and 255 NaN (checked on the device, tests/test_gpu_mx4.py).
__device__ __forceinline__ float mx4_scale(uint32_t e) { return __uint_as_float(e << 23); }

// The gate of the gated products, in 32 bits.  SiLU, g / (1 + e^-g), by h = e^(-|g| / 2): e^-g overflows for gates
// below -88, whose products with a large up 32 bits still hold (gate -89, up 2^100: -2.5e-7), and up times the
// gate may overflow where the result does not (gate -1e20, up 1e20); h does neither.  FINE: expf and a division, for
// results in 32 bits; else the instructions for 2^x and 1 / x, within 2^-16 up to |g| = 100, for results that are
// rounded to bfloat16 (2^-8).  Every kernel goes by that, so the sizes of a product change nothing.
template <bool FINE> __device__ __forceinline__ float mx4_gated(int act, float g, float u) {
  if (act != LLM_ACT_SILU) return llm_gated(act, g, u);
  const float a = fabsf(g), h = FINE ? expf(-0.5f * a) : fast_exp2(-0.72134752f * a), d = 1.0f + h * h;
  const float r = FINE ? 1.0f / d : __builtin_amdgcn_rcpf(d), t = g < 0.f ? h : 1.0f;
  return (u * (t * r)) * (g * t);                          // (neither factor leaves the range before the result does)
}

// Eight codes, widened with their scale; exact (an element has two significant bits), subnormal numbers too, but
// for numbers of 2^128 and more, which only scale bytes of 253 and 254 reach: they become infinities.
__device__ __forceinline__ Frag mx4_widen(uint32_t codes, float scale) {
  union {
    Frag f;
    bf16x2_raw p[4];
  } u;
  u.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0);
  u.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
  u.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2);
  u.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
  return u.f;
}

// C[16 x 16] += A[16 x 128] B[128 x 16], a unit of each; byte OA of `sa` and OB of `sb` are the scales.
template <int OA, int OB>
__device__ __forceinline__ f32x4 mx4_mfma(const uint4& a, uint32_t sa, const uint4& b, uint32_t sb, f32x4 c) {
  const i32x8_raw va = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0};
  const i32x8_raw vb = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(va, vb, c, 4, 4, OA, (int)sa, OB, (int)sb);
}
