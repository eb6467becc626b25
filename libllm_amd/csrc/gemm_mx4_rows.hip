// C[M,N] = X[M,K] * W[N,K]^T for a weight in MXFP4 (mx4.h) and few rows, bound by the one pass over
// W: X in bfloat16 (W's codes are widened to bfloat16, exactly, in front of
// v_mfma_f32_16x16x32_bf16) or in MXFP4 too (v_mfma_scale_f32_16x16x128_f8f6f4 takes both as they
// lie).  Sums in float32, result bfloat16 or float32, or gated over a stacked [gate; up] weight
// (out[m, i] = act(gate_i) * up_i, both still in 32 bits: one rounding).
//
// The waves of a block split K, a run of units of 128 elements each, and every wave goes through its
// run alone: W and X go from memory straight into registers, STAGES units ahead of the arithmetic,
// with no shared memory and no barrier until the waves' sums are added there, in their order.  The
// waves of a block read different elements of X, so sharing them would gain nothing.  Which wave
// adds which unit does not depend on M: an output is the same bits whatever else is in the batch.
#include "mx4.h"

#define MR_WAVES 8           // waves that split K
#define MR_EPI_NONE 0
#define MR_EPI_GATED 1

struct Mx4Args {
  const bf16_t* X;           // rows in bfloat16, ldx elements apart (a multiple of 8, K too), or null:
  const uint4* xc;           // rows in MXFP4
  const uint32_t* xs;
  const uint4* wc;           // W
  const uint32_t* ws;
  const float* bias;         // [N] or null (plain epilogue)
  void* C;
  int M, N, K;               // N: rows of W
  int n_out;                 // columns of C: N, or N / 2 if gated
  int ldx, units, quads, act;
  hipStream_t stream;
};

// Rows of X of a unit, as lane l's B operands.
template <int MT, bool X4> struct RowsOf;
template <int MT> struct RowsOf<MT, false> { Frag f[MT][4]; };
template <int MT> struct RowsOf<MT, true> { uint4 c[MT]; uint32_t s[MT]; };

template <int MT, int RT, int STAGES, int EPI, typename OutT, bool X4>
__global__ __launch_bounds__(MR_WAVES * 64) void gemm_mx4_rows_kernel(Mx4Args a) {
  constexpr int RPR = EPI == MR_EPI_GATED ? 2 : 1;        // tiles of W that make one tile of outputs
  constexpr int OUT_RT = RT / RPR;
  __shared__ __attribute__((aligned(16))) float red[MR_WAVES * RPR * MT * 256];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int r = lane & 15, g = lane >> 4;
  const int out_tile0 = blockIdx.x * OUT_RT, m0 = blockIdx.y * (16 * MT);
  const int out_tiles = (a.n_out + 15) / 16;

  const uint4* wc[RT];
  const uint32_t* ws[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    int t = out_tile0 + rt / RPR;
    if (t > out_tiles - 1) t = out_tiles - 1;             // (not stored)
    if (RPR == 2) t += (rt & 1) * out_tiles;              // up follows gate; n_out is a multiple of 16
    wc[rt] = a.wc + (size_t)t * a.units * 64 + lane;
    ws[rt] = a.ws + (size_t)t * a.quads * 64 + lane;
  }
  const bf16_t* xp[MT];
  bool x_on[MT];
  size_t xt[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int row = m0 + mt * 16 + r;
    x_on[mt] = X4 ? m0 + mt * 16 < a.M : row < a.M;
    xp[mt] = a.X + (size_t)(row < a.M ? row : 0) * a.ldx + g * MX4_BLOCK;
    xt[mt] = (size_t)(m0 / 16 + mt);
  }

  struct Stage {
    uint4 w[RT];
    uint32_t s[RT];
    RowsOf<MT, X4> x;
  };
  auto load = [&](int u, Stage& st) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const u32x4_raw v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_raw*>(wc[rt] + (size_t)u * 64));
      st.w[rt] = make_uint4(v.x, v.y, v.z, v.w);
      st.s[rt] = ws[rt][(size_t)(u >> 2) * 64];
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      if constexpr (X4) {
        st.x.c[mt] = x_on[mt] ? a.xc[(xt[mt] * a.units + u) * 64 + lane] : make_uint4(0u, 0u, 0u, 0u);
        st.x.s[mt] = x_on[mt] ? a.xs[(xt[mt] * a.quads + (u >> 2)) * 64 + lane] : 0u;
      } else {
        const int k = u * MX4_UNIT + g * MX4_BLOCK;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          st.x.f[mt][j] = (x_on[mt] && k + 8 * j < a.K) ? frag_load(xp[mt] + (size_t)u * MX4_UNIT + 8 * j) : frag_zero();
      }
    }
  };
  f32x4 acc[RT][MT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) acc[rt][mt] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto compute = [&](int u, const Stage& st) {
    const int sh = 8 * (u & 3);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      if constexpr (X4) {
        const uint32_t sa = st.s[rt] >> sh;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          acc[rt][mt] = mx4_mfma<0, 0>(st.w[rt], sa, st.x.c[mt], st.x.s[mt] >> sh, acc[rt][mt]);
      } else {
        const float sf = mx4_scale((st.s[rt] >> sh) & 255u);
        const uint32_t w[4] = {st.w[rt].x, st.w[rt].y, st.w[rt].z, st.w[rt].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const Frag f = mx4_widen(w[j], sf);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) acc[rt][mt] = mfma_bf16(f, st.x.f[mt][j], acc[rt][mt]);
        }
      }
    }
  };

  // this wave's run of units
  const int per = (a.units + MR_WAVES - 1) / MR_WAVES;
  const int first = wave * per, last = min(a.units, first + per);
  if (first < last) {
    Stage st[STAGES];
#pragma unroll
    for (int d = 0; d < STAGES; ++d) load(min(first + d, last - 1), st[d]);
    int u = first;
    for (; u + STAGES <= last; u += STAGES) {
#pragma unroll
      for (int d = 0; d < STAGES; ++d) {
        compute(u + d, st[d]);
        load(min(u + d + STAGES, last - 1), st[d]);      // (past the end: the last unit again, unused)
      }
    }
#pragma unroll
    for (int d = 0; d < STAGES - 1; ++d)
      if (u + d < last) compute(u + d, st[d]);
  }

  // ---- the waves' sums, added in order through shared memory, one tile of outputs a round
#pragma unroll
  for (int ort = 0; ort < OUT_RT; ++ort) {
    if (ort > 0) __syncthreads();
#pragma unroll
    for (int j = 0; j < RPR; ++j)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
        *reinterpret_cast<float4*>(red + (((wave * RPR + j) * MT + mt) * 64 + lane) * 4) =
            make_float4(acc[ort * RPR + j][mt][0], acc[ort * RPR + j][mt][1], acc[ort * RPR + j][mt][2],
                        acc[ort * RPR + j][mt][3]);
    __syncthreads();
    if (tid < MT * 64) {
      const int mt = tid >> 6;
      const int m = m0 + mt * 16 + r, n = (out_tile0 + ort) * 16 + 4 * g;
      float v[RPR][4];
#pragma unroll
      for (int j = 0; j < RPR; ++j) {
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < MR_WAVES; ++w) {
          const float4 p = *reinterpret_cast<const float4*>(red + (((w * RPR + j) * MT + mt) * 64 + lane) * 4);
          s.x += p.x; s.y += p.y; s.z += p.z; s.w += p.w;
        }
        v[j][0] = s.x; v[j][1] = s.y; v[j][2] = s.z; v[j][3] = s.w;
      }
      if (m < a.M && n < a.n_out) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (EPI == MR_EPI_GATED) v[0][e] = llm_gated(a.act, v[0][e], v[RPR - 1][e]);
          else if (a.bias != nullptr && n + e < a.n_out) v[0][e] += a.bias[n + e];
        }
        OutT* dst = (OutT*)a.C + (size_t)m * a.n_out + n;
        if (n + 3 < a.n_out && (a.n_out & 3) == 0) {
          Conv4<OutT>::store(dst, make_float4(v[0][0], v[0][1], v[0][2], v[0][3]));
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < a.n_out) Conv<OutT>::store(dst + e, v[0][e]);
        }
      }
    }
  }
}

template <int MT, int RT, int STAGES, int EPI, typename OutT, bool X4>
static int launch_mx4_rows(const Mx4Args& a) {
  constexpr int OUT_RT = EPI == MR_EPI_GATED ? RT / 2 : RT;
  const int tiles = (a.n_out + 15) / 16;
  const dim3 grid((tiles + OUT_RT - 1) / OUT_RT, (a.M + 16 * MT - 1) / (16 * MT));
  if (grid.y > 65535) return LLM_ERR_ARG;
  gemm_mx4_rows_kernel<MT, RT, STAGES, EPI, OutT, X4><<<grid, MR_WAVES * 64, 0, a.stream>>>(a);
  return llm_launch_status();
}

template <int EPI, typename OutT, bool X4>
static int pick_mx4_rows(const Mx4Args& a) {
  if (a.M <= 16) return launch_mx4_rows<1, 2, 4, EPI, OutT, X4>(a);
  if (a.M <= 32) return launch_mx4_rows<2, 2, 2, EPI, OutT, X4>(a);
  return launch_mx4_rows<4, 2, 2, EPI, OutT, X4>(a);
}

template <bool X4>
static int mx4_rows(const Mx4Args& a, int epilogue, int out_dtype) {
  if (epilogue == MR_EPI_NONE) {
    if (out_dtype == LLM_DTYPE_BF16) return pick_mx4_rows<MR_EPI_NONE, bf16_t, X4>(a);
    if (out_dtype == LLM_DTYPE_F32) return pick_mx4_rows<MR_EPI_NONE, float, X4>(a);
  } else if (epilogue == MR_EPI_GATED && out_dtype == LLM_DTYPE_BF16) {
    return pick_mx4_rows<MR_EPI_GATED, bf16_t, X4>(a);
  }
  return LLM_ERR_ARG;
}

// W [N, K] as mx4.h lays it out.  X: bfloat16 rows ldx apart (K and ldx multiples of 8, 16-byte
// aligned) with xs null, or codes with their scales in xs.  epilogue 0: C [M, N] of out_dtype, plus
// bias[n] if not null; 1 | act << 4: C [M, N / 2] in bfloat16, the gate through an activation of
// common.h, N / 2 a multiple of 16.
extern "C" int llm_gemm_mx4_rows(const void* X, const void* xs, int ldx, const void* wc, const void* ws,
                                 const float* bias, void* C, int epilogue, int out_dtype, int M, int N, int K,
                                 hipStream_t stream) {
  if (M <= 0) return LLM_OK;
  const int act = epilogue >> 4;
  epilogue &= 15;
  if (N <= 0 || K <= 0 || act < 0 || act >= LLM_ACT_COUNT || (epilogue != MR_EPI_GATED && act != 0)) return LLM_ERR_ARG;
  if (X == nullptr || wc == nullptr || ws == nullptr || C == nullptr) return LLM_ERR_ARG;
  if ((((uintptr_t)X) | ((uintptr_t)wc) | ((uintptr_t)ws) | ((uintptr_t)C) | ((uintptr_t)xs)) & 15) return LLM_ERR_ARG;
  if (xs == nullptr && (ldx < K || (ldx & 7) || (K & 7))) return LLM_ERR_ARG;
  if (epilogue == MR_EPI_GATED && ((N & 31) || bias != nullptr)) return LLM_ERR_ARG;
  Mx4Args a{};
  a.X = (const bf16_t*)X;
  a.xc = (const uint4*)X;
  a.xs = (const uint32_t*)xs;
  a.wc = (const uint4*)wc;
  a.ws = (const uint32_t*)ws;
  a.bias = bias;
  a.C = C;
  a.M = M;
  a.N = N;
  a.K = K;
  a.n_out = epilogue == MR_EPI_GATED ? N / 2 : N;
  a.ldx = ldx;
  a.units = mx4_units(K);
  a.quads = mx4_quads(K);
  a.act = act;
  a.stream = stream;
  return xs == nullptr ? mx4_rows<false>(a, epilogue, out_dtype) : mx4_rows<true>(a, epilogue, out_dtype);
}
