// C[M,N] = X[M,K] * W[N,K]^T for a weight in MXFP4 (mx4.h) and few rows, bound by the one pass over
// W: X in bfloat16 (W's codes are widened to bfloat16, exactly, in front of
// v_mfma_f32_16x16x32_bf16) or in MXFP4 too (v_mfma_scale_f32_16x16x128_f8f6f4 takes both as they
// lie).  Sums in float32, result bfloat16 or float32, or gated over a stacked [gate; up] weight
// (out[m, i] = act(gate_i) * up_i, both still in 32 bits: one rounding), or added into the residual
// stream, or rotated and written to the cache.  With rows in bfloat16 an RMS norm between two products
// needs no kernel of its own up to 16 rows, as in the product for few rows with bfloat16 weights (there
// is why): the product that adds into the stream prepares it, the product behind it multiplies its sums
// by the row's scale.
//
// The waves of a block split K, a run of units of 128 elements each, and every wave goes through its
// run alone, with no barrier until the waves' sums are added at the end, in their order.  W goes from
// memory straight into registers, STAGES units ahead of the arithmetic.  Rows of X in bfloat16 are
// loaded as they lie, four rows by 256 bytes an instruction (whole lines), also STAGES ahead, and
// turned into the matrix cores' operand through 4 KiB of shared memory that only this wave uses;
// read straight from memory in operand order, 16 rows by four pieces of 16 bytes far apart, they
// bounded the kernel (8 rows, K 14,336, 4,096 outputs: 18.0 us).  The waves of a block read
// different elements of X, so sharing them would gain nothing.  Which wave adds which unit does not
// depend on M: an output is the same bits whatever else is in the batch.
#include "mx4.h"
#include "row_epilogue.h"

#define MR_EPI_NONE 0
#define MR_EPI_GATED 1
#define MR_EPI_ACCUM 2
#define MR_EPI_ROPE 3

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
  int ldx, units, quads, act;   // units: those that hold elements of K
  hipStream_t stream;
  const float* next_w;       // accumulating: weight [N] of the norm that reads the stream next, or null
  bf16_t* raw;               //   out [M, N]: the new stream times next_w
  float* ssq_out;            //   out [M, N / 16]: sums of squares of the new stream over tiles of 16 columns
  const float* ssq_in;       // [M, K / 16]: such sums for the rows of X, which still lack their scale; or null
  float eps;
  RowRope rope;
};

// WAVES: waves that split K; MT: tiles of 16 rows of X; XQ: quarters of a tile of which rows exist (4 unless MT is 1);
// RT: tiles of W a wave; STAGES: units in flight.
template <int WAVES, int MT, int XQ, int RT, int STAGES, int EPI, bool NORM, typename OutT, bool X4>
__global__ __launch_bounds__(WAVES * 64) void gemm_mx4_rows_kernel(Mx4Args a) {
  constexpr int RPR = EPI == MR_EPI_GATED ? 2 : 1;        // tiles of W that make one tile of outputs
  constexpr int OUT_RT = RT / RPR;
  constexpr int XL = X4 ? MT : (MT - 1) * 4 + XQ;         // loads of rows of X a unit
  constexpr int WAVE_B = X4 ? RPR * MT * 1024 : 4096 * MT;
  __shared__ __attribute__((aligned(16))) unsigned char lds[WAVES * WAVE_B];
  float* red = reinterpret_cast<float*>(lds);
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int r = lane & 15, g = lane >> 4;
  __shared__ float s_scale[16];                           // a row's rsqrt(mean(x^2) + eps) where X lacks it
  const int out_tile0 = blockIdx.x * OUT_RT, m0 = blockIdx.y * (16 * MT);
  const int out_tiles = (a.n_out + 15) / 16;
  unsigned char* mine = lds + wave * WAVE_B;

  const uint4* wc[RT];
  const uint32_t* ws[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    int t = out_tile0 + rt / RPR;
    if (t > out_tiles - 1) t = out_tiles - 1;             // (not stored)
    if (RPR == 2) t += (rt & 1) * out_tiles;              // up follows gate; n_out is a multiple of 16
    wc[rt] = a.wc + (size_t)t * a.quads * 256 + lane;
    ws[rt] = a.ws + (size_t)t * a.quads * 64 + lane;
  }
  // Rows past the end are read as the last row (bfloat16) or tile (MXFP4); their sums are not stored.
  const bf16_t* xp[XL];
  const uint4* xc[MT];
  const uint32_t* xs[MT];
#pragma unroll
  for (int i = 0; i < XL; ++i) xp[i] = a.X + (size_t)min(m0 + i * 4 + g, a.M - 1) * a.ldx;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const size_t t = min(m0 / 16 + mt, (a.M - 1) / 16);
    xc[mt] = a.xc + t * a.quads * 256 + lane;
    xs[mt] = a.xs + t * a.quads * 64 + lane;
  }

  struct Stage {
    uint4 w[RT], x[XL];
    uint32_t s[RT], xs[X4 ? MT : 1];
  };
  auto load = [&](int u, Stage& st) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const u32x4_raw v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_raw*>(wc[rt] + (size_t)u * 64));
      st.w[rt] = make_uint4(v.x, v.y, v.z, v.w);
      st.s[rt] = ws[rt][(size_t)(u >> 2) * 64];
    }
    if constexpr (X4) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        st.x[mt] = xc[mt][(size_t)u * 64];
        st.xs[mt] = xs[mt][(size_t)(u >> 2) * 64];
      }
    } else {
      const int k = u * MX4_UNIT + r * 8;                 // piece r of a row's 256 bytes
      const int at = k < a.K ? k : 0;
#pragma unroll
      for (int i = 0; i < XL; ++i) st.x[i] = *reinterpret_cast<const uint4*>(xp[i] + at);
    }
  };
  f32x4 acc[RT][MT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) acc[rt][mt] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto compute = [&](int u, Stage& st) {
    const int sh = 8 * (u & 3);
    if constexpr (X4) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          acc[rt][mt] = mx4_mfma<0, 0>(st.w[rt], st.s[rt] >> sh, st.x[mt], st.xs[mt] >> sh, acc[rt][mt]);
    } else {
      // past K the rows are zero, as W is there (a load past it has read elements that may be no numbers;
      // a select at the load would be a branch, and the loads in flight no longer counted)
      if ((u + 1) * MX4_UNIT > a.K) {
        const uint32_t keep = u * MX4_UNIT + r * 8 < a.K ? 0xffffffffu : 0u;
#pragma unroll
        for (int i = 0; i < XL; ++i)
          st.x[i] = make_uint4(st.x[i].x & keep, st.x[i].y & keep, st.x[i].z & keep, st.x[i].w & keep);
      }
      // piece p of row m of a tile lies at m * 256 + (p ^ m) * 16: rows of a read and pieces of a
      // write fall into different banks.  A wave's accesses to shared memory run in order; the empty
      // statements keep the compiler from moving one lane's read over another lane's write.
#pragma unroll
      for (int i = 0; i < XL; ++i) {
        const int m = (i & 3) * 4 + g;
        *reinterpret_cast<uint4*>(mine + (i >> 2) * 4096 + m * 256 + ((r ^ m) * 16)) = st.x[i];
      }
      asm volatile("" ::: "memory");
      Frag x[4][MT];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          x[j][mt].u = *reinterpret_cast<const uint4*>(mine + mt * 4096 + r * 256 + (((g * 4 + j) ^ r) * 16));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const uint32_t w[4] = {st.w[rt].x, st.w[rt].y, st.w[rt].z, st.w[rt].w};
          const Frag f = mx4_widen(w[j], mx4_scale((st.s[rt] >> sh) & 255u));
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) acc[rt][mt] = mfma_bf16(f, x[j][mt], acc[rt][mt]);
        }
      }
      asm volatile("" ::: "memory");
    }
  };

  // this wave's run of units
  const int per = (a.units + WAVES - 1) / WAVES;
  const int first = wave * per, last = min(a.units, first + per);
  // What the epilogue needs from memory beside the sums is asked for in front of the first loads: the wave
  // of a row tile finishes its columns 4 g .. 4 g + 3, 16 apart a round.  No branch here: one between the
  // first loads and the loop makes the compiler hold everything in flight twice.
  const int e_m = m0 + wave * 16 + r, e_n0 = out_tile0 * 16 + 4 * g;
  const int e_row = min(e_m, a.M - 1);                     // (a row that exists; what belongs to another is not stored)
  RopeSteps<EPI == MR_EPI_ROPE ? OUT_RT : 1> e_rope;
  float e_prev[EPI == MR_EPI_ACCUM ? OUT_RT : 1][4], e_nw[EPI == MR_EPI_ACCUM && NORM ? OUT_RT : 1][4];
  if constexpr (EPI == MR_EPI_ROPE) e_rope.first(a.rope, e_row);
  if constexpr (EPI == MR_EPI_ACCUM) {
#pragma unroll
    for (int ort = 0; ort < OUT_RT; ++ort)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = min(e_n0 + ort * 16 + e, a.n_out - 1);
        e_prev[ort][e] = ((const float*)a.C)[(size_t)e_row * a.n_out + n];
        if constexpr (NORM) e_nw[ort][e] = a.next_w[n];
      }
  }
  // The sums of squares of a row of X that still lacks its scale: TPR neighbouring threads a row.
  constexpr int TPR = WAVES * 4, SS_AHEAD = 8;
  static_assert(TPR <= 64, "the threads of a row lie in one wave");
  constexpr bool SCALES = NORM && EPI != MR_EPI_ACCUM;
  static_assert(!NORM || (MT == 1 && !X4), "norms are folded for up to 16 rows in bfloat16");
  float e_ss[SS_AHEAD];
  const int ss_row = tid / TPR, ss_part = tid % TPR, parts_in = a.K / 16;
  const size_t ss_at = (size_t)min(ss_row, a.M - 1) * parts_in;
  if constexpr (SCALES) {
#pragma unroll
    for (int i = 0; i < SS_AHEAD; ++i) {
      const int p = ss_part + i * TPR;
      const float q = a.ssq_in[ss_at + min(p, parts_in - 1)];
      e_ss[i] = p < parts_in ? q : 0.f;
    }
  }
  Stage st[STAGES];
#pragma unroll
  for (int d = 0; d < STAGES; ++d) load(min(first + d, a.units - 1), st[d]);      // (a wave may have none)
  if constexpr (EPI == MR_EPI_ROPE) e_rope.second(a.rope, e_n0);
  int u = first;
  for (; u + STAGES <= last; u += STAGES) {
#pragma unroll
    for (int d = 0; d < STAGES; ++d) {
      compute(u + d, st[d]);
      load(min(u + d + STAGES, last - 1), st[d]);        // (past the end: the last unit again, unused)
    }
  }
#pragma unroll
  for (int d = 0; d < STAGES - 1; ++d)
    if (u + d < last) compute(u + d, st[d]);
  if constexpr (EPI == MR_EPI_ROPE) e_rope.third(a.rope);
  if constexpr (SCALES) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < SS_AHEAD; ++i) ss += e_ss[i];
    for (int p = ss_part + SS_AHEAD * TPR; p < parts_in; p += TPR) ss += a.ssq_in[ss_at + p];      // wider rows
#pragma unroll
    for (int off = TPR / 2; off >= 1; off >>= 1) ss += __shfl_xor(ss, off, 64);
    if (ss_part == 0) s_scale[ss_row] = rsqrtf(ss / (float)a.K + a.eps);      // read behind the next barrier
  }

  // ---- the waves' sums, added in order through shared memory (a wave writes where its rows of X
  // lay), one tile of outputs a round
  constexpr int RED = WAVE_B / 4;
#pragma unroll
  for (int ort = 0; ort < OUT_RT; ++ort) {
    if (ort > 0) __syncthreads();
#pragma unroll
    for (int j = 0; j < RPR; ++j)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
        *reinterpret_cast<float4*>(red + wave * RED + ((j * MT + mt) * 64 + lane) * 4) =
            make_float4(acc[ort * RPR + j][mt][0], acc[ort * RPR + j][mt][1], acc[ort * RPR + j][mt][2],
                        acc[ort * RPR + j][mt][3]);
    __syncthreads();
    if (wave < MT) {
      const int mt = wave, m = e_m, n = e_n0 + ort * 16;
      float v[RPR][4];
#pragma unroll
      for (int j = 0; j < RPR; ++j) {
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8                                          // (sixteen at once would not fit in the registers)
        for (int w = 0; w < WAVES; ++w) {
          const float4 p = *reinterpret_cast<const float4*>(red + w * RED + ((j * MT + mt) * 64 + lane) * 4);
          s.x += p.x; s.y += p.y; s.z += p.z; s.w += p.w;
        }
        v[j][0] = s.x; v[j][1] = s.y; v[j][2] = s.z; v[j][3] = s.w;
        if constexpr (SCALES) {
          const float sc = s_scale[r];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[j][e] *= sc;
        }
      }
      const bool on = m < a.M && n < a.n_out;
      if constexpr (EPI == MR_EPI_ROPE) {
        if (on) rope_store<OUT_RT>(a.rope, e_rope, ort, v[0], m, n, (bf16_t*)a.C);
        continue;
      }
      if constexpr (EPI == MR_EPI_ACCUM && NORM) {
        norm_store(on, v[0], e_prev[ort], e_nw[ort], m, n, a.n_out, g, (float*)a.C, a.raw, a.ssq_out);
        continue;
      }
      if (on) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (EPI == MR_EPI_GATED) v[0][e] = mx4_gated<sizeof(OutT) == 4>(a.act, v[0][e], v[RPR - 1][e]);
          else if (EPI == MR_EPI_ACCUM) v[0][e] += e_prev[ort][e];
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

template <int WAVES, int MT, int XQ, int RT, int STAGES, int EPI, bool NORM, typename OutT, bool X4>
static int launch_mx4_rows(const Mx4Args& a) {
  constexpr int OUT_RT = EPI == MR_EPI_GATED ? RT / 2 : RT;
  const int tiles = (a.n_out + 15) / 16;
  const dim3 grid((tiles + OUT_RT - 1) / OUT_RT, (a.M + 16 * MT - 1) / (16 * MT));
  if (grid.y > 65535) return LLM_ERR_ARG;
  gemm_mx4_rows_kernel<WAVES, MT, XQ, RT, STAGES, EPI, NORM, OutT, X4><<<grid, WAVES * 64, 0, a.stream>>>(a);
  return llm_launch_status();
}

// How many waves split K depends on W alone (an output's sum does not change with the batch): 16
// where there are tiles of outputs for half of the compute units at most, 8 up to one a unit, else 4,
// whose longer runs overlap better (us, 4 / 8 / 16 waves: 2,048 x 2,048 by 16 rows 4.6 / 4.6 / 3.9;
// 14,336 x 4,096 by one row 9.7 / 8.6 / 8.8; 4,096 x 6,144 by 16 rows 9.6 / 11.6 / 11.2; gate and up
// of 4,096 x 14,336 by 8 rows 20.2 / 26.1 / 28.5).  Where several blocks fall to a unit, few registers
// count for more than units in flight, since then they run at once: 3 units, from 9 rows on 2, where
// there are tiles for three blocks a unit 1 (gate and up of 4,096 x 14,336, us by 8 / 16 rows: 4 units
// 19.5 / 22.7, 3 units 16.7 / 21.0).  From 9 rows on a wave then takes two tiles of outputs, which
// halves what a block reads of X (4,096 x 6,144 by 16 rows, 2 units: 7.1 us against 8.3 by one tile; that
// gate and up by 16 / 32 rows, 1 unit: 17.6 / 22.7 against 21.0 / 27.9); rows in MXFP4, a quarter of the
// bytes, only with tiles for three blocks (4,096 x 16,384 by 16 rows 9.5 against 10.3).
template <int MT, int XQ, int EPI, bool NORM, typename OutT, bool X4>
static int pick_mx4_tiles(const Mx4Args& a) {
  constexpr int ONE = EPI == MR_EPI_GATED ? 2 : 1;
  constexpr bool MANY = X4 || XQ == 4;                    // from 9 rows on
  const int tiles = (a.n_out + 15) / 16, units = llm_compute_units();
  if (tiles <= units / 2) return launch_mx4_rows<16, MT, XQ, ONE, MT == 1 ? 2 : 1, EPI, NORM, OutT, X4>(a);
  if (tiles <= units) return launch_mx4_rows<8, MT, XQ, ONE, MT == 1 ? 3 : 2, EPI, NORM, OutT, X4>(a);
  if constexpr (MANY)
    if (tiles >= 3 * units) return launch_mx4_rows<4, MT, XQ, 2 * ONE, X4 ? 2 : 1, EPI, NORM, OutT, X4>(a);
  return launch_mx4_rows<4, MT, XQ, MANY && !X4 ? 2 * ONE : ONE, MANY ? 2 : 3, EPI, NORM, OutT, X4>(a);
}

template <int EPI, bool NORM, typename OutT, bool X4>
static int pick_mx4_rows(const Mx4Args& a) {
  if constexpr (!X4) {
    if (a.M <= 4) return pick_mx4_tiles<1, 1, EPI, NORM, OutT, X4>(a);
    if (a.M <= 8) return pick_mx4_tiles<1, 2, EPI, NORM, OutT, X4>(a);
  }
  if (a.M <= 16) return pick_mx4_tiles<1, 4, EPI, NORM, OutT, X4>(a);
  if constexpr (!NORM) {
    // 17 to 32 rows of a weight with few tiles in two slabs of 16: blocks for twice as many units (2,048 x
    // 2,048 by 32 rows: 4.0 us against 5.4)
    if (a.M <= 32 && (a.n_out + 15) / 16 <= llm_compute_units() / 2) return pick_mx4_tiles<1, 4, EPI, NORM, OutT, X4>(a);
    return pick_mx4_tiles<2, 4, EPI, NORM, OutT, X4>(a);
  }
  return LLM_ERR_ARG;
}

template <bool X4>
static int mx4_rows(const Mx4Args& a, int epilogue, int out_dtype) {
#define MR_PICK(EPI, T)                                                                              \
  do {                                                                                               \
    if constexpr (!X4)                                                                               \
      if (a.next_w != nullptr || a.ssq_in != nullptr) return pick_mx4_rows<EPI, true, T, X4>(a);     \
    return pick_mx4_rows<EPI, false, T, X4>(a);                                                      \
  } while (0)
  if (epilogue == MR_EPI_NONE) {
    if (out_dtype == LLM_DTYPE_BF16) MR_PICK(MR_EPI_NONE, bf16_t);
    if (out_dtype == LLM_DTYPE_F32) MR_PICK(MR_EPI_NONE, float);
  } else if (epilogue == MR_EPI_GATED && out_dtype == LLM_DTYPE_BF16) {
    MR_PICK(MR_EPI_GATED, bf16_t);
  } else if (epilogue == MR_EPI_ACCUM && out_dtype == LLM_DTYPE_F32) {
    if constexpr (!X4) MR_PICK(MR_EPI_ACCUM, float);
  }
#undef MR_PICK
  return LLM_ERR_ARG;
}

// W [N, K] as mx4.h lays it out.  X: bfloat16 rows ldx apart (K and ldx multiples of 8, 16-byte
// aligned) with xs null, or codes with their scales in xs.  epilogue 0: C [M, N] of out_dtype, plus
// bias[n] if not null; 1 | act << 4: C [M, N / 2] in bfloat16, the gate through an activation of
// common.h, N / 2 a multiple of 16; 2 (bfloat16 rows): added into the float32 C [M, N].
// Around an RMS norm without a kernel of its own (bfloat16 rows, M at most 16; see gemm_skinny.hip):
// epilogue 2 with next_w (N a multiple of 16): beside adding, raw [M, N] = bfloat16(C * next_w) and
// ssq_out [M, N / 16] are written; epilogue 0 or 1 with ssq_in [M, K / 16] (K a multiple of 16): the sums
// are multiplied by rsqrt(sum(ssq_in[m]) / K + eps) first.
extern "C" int llm_gemm_mx4_rows(const void* X, const void* xs, int ldx, const void* wc, const void* ws,
                                 const float* bias, void* C, int epilogue, int out_dtype, int M, int N, int K,
                                 const float* next_w, void* raw, float* ssq_out, const float* ssq_in, float eps,
                                 hipStream_t stream) {
  if (M <= 0) return LLM_OK;
  const int act = epilogue >> 4;
  epilogue &= 15;
  if (N <= 0 || K <= 0 || act < 0 || act >= LLM_ACT_COUNT || (epilogue != MR_EPI_GATED && act != 0)) return LLM_ERR_ARG;
  if (X == nullptr || wc == nullptr || ws == nullptr || C == nullptr) return LLM_ERR_ARG;
  if ((((uintptr_t)X) | ((uintptr_t)wc) | ((uintptr_t)ws) | ((uintptr_t)C) | ((uintptr_t)xs)) & 15) return LLM_ERR_ARG;
  if (xs == nullptr && (ldx < K || (ldx & 7) || (K & 7))) return LLM_ERR_ARG;
  if (epilogue == MR_EPI_GATED && (N & 31)) return LLM_ERR_ARG;
  if (epilogue != MR_EPI_NONE && bias != nullptr) return LLM_ERR_ARG;
  if (next_w != nullptr && (epilogue != MR_EPI_ACCUM || M > 16 || (N & 15) || raw == nullptr || ssq_out == nullptr ||
                            (((uintptr_t)raw) & 15)))
    return LLM_ERR_ARG;
  if (ssq_in != nullptr && (epilogue == MR_EPI_ACCUM || xs != nullptr || M > 16 || (K & 15) || !(eps >= 0.f))) return LLM_ERR_ARG;
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
  a.next_w = next_w;
  a.raw = (bf16_t*)raw;
  a.ssq_out = ssq_out;
  a.ssq_in = ssq_in;
  a.eps = eps;
  return xs == nullptr ? mx4_rows<false>(a, epilogue, out_dtype) : mx4_rows<true>(a, epilogue, out_dtype);
}

// The stacked q|k|v projection with the rotary epilogue: rotated q as bfloat16 [M, n_heads * hd] to
// q_out, k and v to the cache if write_kv.  W has (n_heads + 2 n_kv) * hd rows with write_kv, else n_heads
// * hd; hd a multiple of 16, rot_dim even.  ssq_in as above.
extern "C" int llm_gemm_mx4_rows_rope(const void* X, int ldx, const void* wc, const void* ws, const float* bias,
                                      void* q_out, int M, int K, int n_heads, int n_kv, int hd, const float* cos_t,
                                      const float* sin_t, int rot_dim, const int* tok_pos, const int* tok_seq,
                                      const int* seq_slot, const int* table, int table_stride, void* k_pages,
                                      void* v_pages, int page_size, int write_kv, const float* ssq_in, float eps,
                                      hipStream_t stream) {
  if (M <= 0) return LLM_OK;
  if (ssq_in != nullptr && (M > 16 || (K & 15) || !(eps >= 0.f))) return LLM_ERR_ARG;
  if (K <= 0 || (K & 7) || ldx < K || (ldx & 7) || n_heads <= 0 || n_kv < 0 || hd <= 0 || (hd & 15) || rot_dim < 0 ||
      rot_dim > hd || (rot_dim & 1) || page_size != LLM_PAGE)
    return LLM_ERR_ARG;
  if (X == nullptr || wc == nullptr || ws == nullptr || q_out == nullptr || tok_pos == nullptr) return LLM_ERR_ARG;
  if ((((uintptr_t)X) | ((uintptr_t)wc) | ((uintptr_t)ws) | ((uintptr_t)q_out)) & 15) return LLM_ERR_ARG;
  if (rot_dim > 0 && (cos_t == nullptr || sin_t == nullptr)) return LLM_ERR_ARG;
  if (write_kv && (!k_pages || !v_pages || !table || !seq_slot || !tok_seq || n_kv <= 0 ||
                   ((((uintptr_t)k_pages) | ((uintptr_t)v_pages)) & 7)))
    return LLM_ERR_ARG;
  Mx4Args a{};
  a.X = (const bf16_t*)X;
  a.wc = (const uint4*)wc;
  a.ws = (const uint32_t*)ws;
  a.C = q_out;
  a.M = M;
  a.N = (n_heads + (write_kv ? 2 * n_kv : 0)) * hd;
  a.K = K;
  a.n_out = a.N;
  a.ldx = ldx;
  a.units = mx4_units(K);
  a.quads = mx4_quads(K);
  a.stream = stream;
  a.ssq_in = ssq_in;
  a.eps = eps;
  a.rope = RowRope{bias, cos_t, sin_t, tok_pos, tok_seq, seq_slot, table, (bf16_t*)k_pages, (bf16_t*)v_pages,
                   table_stride, n_heads, n_kv, hd, rot_dim, write_kv};
  if (ssq_in != nullptr) return pick_mx4_rows<MR_EPI_ROPE, true, bf16_t, false>(a);
  return pick_mx4_rows<MR_EPI_ROPE, false, bf16_t, false>(a);
}
