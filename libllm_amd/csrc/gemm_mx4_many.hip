// C[M,N] = X[M,K] * W[N,K]^T for a weight in MXFP4 (mx4.h) and many rows, bound by the matrix cores
// and by what a compute unit can pull into its shared memory.  Rows in bfloat16: W's codes are widened
// to bfloat16 in front of v_mfma_f32_16x16x32_bf16, exactly, so the result is that of a bfloat16
// product with W's numbers.  Rows in MXFP4: v_mfma_scale_f32_16x16x128_f8f6f4, four times the
// arithmetic an instruction.  Sums in float32; result bfloat16 or float32, or gated over a stacked
// [gate; up] weight (out[m, i] = act(gate_i) * up_i, in 32 bits until the one rounding).
//
// A block of waves, WM along the rows of X by WN along those of W, owns 16 WM MTW rows of X by
// 16 WN NTW rows of W (gated: half of them gate, half the up rows of the same columns); W is the A
// operand, so that a lane ends with four consecutive columns of one row of C.  K goes by in tiles:
// 128 elements (bfloat16, four steps of 32) or 256 (MXFP4, two steps of 128).  X's tiles go from
// memory straight into LDS (global_load_lds_dwordx4), two to six buffers by form.  In bfloat16 a row of
// a tile is 256 bytes in 16 pieces; piece p of row r lies at p ^ (r & 15), so that the 16 rows a fragment
// read touches fall into different banks.  In MXFP4 the tiles lie in lane order as they come.  W's codes
// are a quarter of X's bytes: with rows in bfloat16 and two buffers they stay in registers, read straight
// from the caches by every wave that needs them, one tile of K ahead; with more buffers, and with rows in
// MXFP4, they go through LDS like X's, and the scales too, four units at a time.
//
// The fragments of a step are read into registers one step (EARLY: two) ahead of the matrix instructions
// that use them, dealt out between those; the barrier of a tile lies in front of its last step, whose
// fragments every wave has by then: behind it the loads of a later tile go out into the buffer that
// is left, and the first fragments of the next tile are read.
#include "mx4.h"

#include <type_traits>

// The kernel is written in lambdas over fixed arrays of registers: each has to go into the kernel whole.
#define MM_INLINE __attribute__((always_inline))

#define MM_EPI_NONE 0
#define MM_EPI_GATED 1

struct Mx4ManyArgs {
  const bf16_t* X;           // rows in bfloat16, ldx apart; K and ldx multiples of 128
  const uint8_t* xc;         // or rows in MXFP4
  const uint8_t* xs;
  const uint8_t* wc;
  const uint8_t* ws;
  const float* bias;         // [N] or null (plain epilogue)
  void* C;
  int M, N, n_out;
  int ldx, units, quads, act;
  int m_tiles, n_tiles;      // blocks along X and W
  int slice_quads;           // quads of K a slice (blockIdx.y counts them); one slice has them all
  hipStream_t stream;
};

template <int N, typename F> __device__ __forceinline__ void each(F&& f) {
  if constexpr (N > 0) {
    each<N - 1>(f);
    f(std::integral_constant<int, N - 1>{});
  }
}

// 16 bytes a lane from base + off into LDS, in lane order from `lds` on, without registers in
// between.  Written in assembly: the compiler would make every read of LDS wait for all of them (it
// cannot tell that they fill the other buffer).  It does not count them either: the kernel waits
// for them itself, before the barrier that hands a buffer over.  (The instruction takes its place in
// LDS from M0, which is put back: the compiler need not know.)
__device__ __forceinline__ void lds_fill(uint32_t lds, const void* base, uint32_t off) {
  uint32_t m0_was;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3\n\ts_mov_b32 m0, %0"
               : "=&s"(m0_was) : "s"(lds), "v"(off), "s"(base) : "memory");
}

// Sizes of a form.  A tile of K is UPT units of 128 elements, NBUF of them are held in LDS.  EARLY: with
// few waves a unit nothing covers the latency of LDS; fragments are then read two steps ahead (into a second
// set) instead of one, and the barrier of a tile lies a step earlier.  A buffer is filled again a tile
// later than it could be: its reads are long over by then, and the barrier need not wait for those
// under way.
template <bool X4, int NBUF, bool EARLY, int WM, int WN, int MTW, int NTW>
struct ManyShape {
  static constexpr int UPT = X4 ? 2 : 1;
  static constexpr int BM = WM * MTW * 16, BNT = WN * NTW;          // rows of X, tiles of W a block
  static constexpr bool WL = X4 || NBUF > 2;                        // W's codes and scales go through LDS
  static constexpr int XB = X4 ? BM * 64 * UPT : BM * 256;          // bytes of X's tile of K
  static constexpr int BUF = XB + (X4 ? BNT * 1024 * UPT : WL ? BNT * 1024 : 0);
  static constexpr int TPQ = 4 / UPT;                               // tiles of K a quad
  static constexpr int FAR = EARLY ? NBUF - 1 : NBUF;               // tiles from the one at work to the one asked for
  static constexpr int STILES = X4 ? BM / 16 + BNT : WL ? BNT : 0;  // tiles whose scales go through LDS: W's, then X's
  static constexpr int SB = STILES * 256, NSB = (FAR + TPQ - 1) / TPQ;      // scales of a quad, quads held
  static constexpr int BYTES = NBUF * BUF + NSB * SB;
};

template <bool X4, int NBUF, bool EARLY, int WM, int WN, int MTW, int NTW, int EPI, typename OutT>
__global__ __launch_bounds__(WM * WN * 64) void gemm_mx4_many_kernel(Mx4ManyArgs a) {
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  typedef ManyShape<X4, NBUF, EARLY, WM, WN, MTW, NTW> Shape;
  constexpr int NW = WM * WN;
  constexpr int BM = Shape::BM, BNT = Shape::BNT, XB = Shape::XB, BUF = Shape::BUF, STILES = Shape::STILES, SB = Shape::SB;
  constexpr int FAR = Shape::FAR, NSB = Shape::NSB, TPQ = Shape::TPQ, UPT = Shape::UPT;
  constexpr bool WL = Shape::WL;
  constexpr int STEPS = X4 ? UPT : 4;                       // steps of matrix instructions a tile of K
  constexpr int AHEAD = EARLY ? 2 : 1, BSTEP = STEPS - AHEAD;
  constexpr int TURNS = WL && TPQ > 2 ? TPQ : 2;            // rounds after which sets of registers and bytes of scales repeat
  constexpr int XF = XB / 1024 / NW, FILLS = BUF / 1024 / NW;       // loads of 1 KiB a wave and tile: X's, all
  constexpr int XT = UPT * 1024;                            // bytes of a row tile of X, or a tile of W, in MXFP4
  static_assert(XB % (1024 * NW) == 0 && BUF % (1024 * NW) == 0, "every wave fills as much");
  static_assert(STEPS >= AHEAD && (STEPS * TURNS) % 2 == 0 && TURNS % TPQ == 0 || !WL, "the sets repeat");
  constexpr bool GATED = EPI == MM_EPI_GATED;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int r = lane & 15, g = lane >> 4;
  const int wm = wave % WM, wn = wave / WM;

  // blocks i, i + 8, ... share a chiplet: a chiplet takes every eighth tile of W rows and, at a
  // time, a band of 8 tiles of X rows
  const int xcd = blockIdx.x & 7, jb = blockIdx.x >> 3;
  const int n_per = (a.n_tiles + 7) >> 3;
  const int band = jb / (8 * n_per), jj = jb - band * (8 * n_per);
  const int band_rows = min(a.m_tiles - band * 8, 8);
  const int mt_blk = band * 8 + jj % band_rows, nt_blk = (jj / band_rows) * 8 + xcd;
  if (nt_blk >= a.n_tiles || jj >= band_rows * n_per) return;
  const int m0 = mt_blk * BM;
  const int out_tiles = (a.n_out + 15) / 16;

  // tile of W that is number t of this block (past the end the last one; its sums are not stored)
  auto w_tile = [&](int t) MM_INLINE {
    if (GATED) return min(nt_blk * (BNT / 2) + t % (BNT / 2), out_tiles - 1) + (t / (BNT / 2)) * out_tiles;
    return min(nt_blk * BNT + t, out_tiles - 1);
  };
  // number within the block of tile nt of this wave: gated, its gate tiles and then its up tiles
  auto wave_tile = [&](int nt) MM_INLINE {
    return GATED ? (nt / (NTW / 2)) * (BNT / 2) + wn * (NTW / 2) + nt % (NTW / 2) : wn * NTW + nt;
  };
  const size_t c_tile = (size_t)a.quads * 4096, s_tile = (size_t)a.quads * 256;
  // K may be a slice, a run of whole quads: everything begins that far into its rows, and the sums go
  // to a matrix of the slice's own (plain epilogue in float32), to be added in order by whoever reads them
  const int q0 = blockIdx.y * a.slice_quads;
  const int units = min(a.units - 4 * q0, 4 * a.slice_quads), quads = min(a.quads - q0, a.slice_quads);
  a.X += (size_t)q0 * 512;
  a.xc += (size_t)q0 * 4096;
  a.wc += (size_t)q0 * 4096;
  a.xs += (size_t)q0 * 256;
  a.ws += (size_t)q0 * 256;
  a.C = (OutT*)a.C + (size_t)blockIdx.y * a.M * a.n_out;

  // ---- what this wave fills, and where from
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds;
  static_assert(X4 || NW % 4 == 0, "the rows a wave fills lie a multiple of 16 apart");
  const uint32_t lane16 = lane * 16, lane4 = lane * 4;
  const uint8_t* fill_base[FILLS];
  int fill_row = 0;
  uint32_t fill_piece = 0;
#pragma unroll
  for (int p = 0; p < FILLS; ++p) {
    const int c = p * NW + wave;                            // which KiB of the buffer
    if (X4) {                                               // (tile, unit) of X, then of W
      const int t = c / UPT;
      fill_base[p] = (p < XF ? a.xc + (size_t)min(m0 / 16 + t, (a.M - 1) / 16) * c_tile
                             : a.wc + (size_t)w_tile(t - BM / 16) * c_tile) + (c % UPT) * 1024;
    } else {                                                // four rows of X; a tile of W
      fill_base[p] = p < XF ? (const uint8_t*)(a.X + (size_t)m0 * a.ldx) : a.wc + (size_t)w_tile(c - XB / 1024) * c_tile;
    }
  }
  if constexpr (!X4) {
    fill_row = wave * 4 + g;
    fill_piece = (r ^ (fill_row & 15)) * 16;
  }
  // scales of a quad: a KiB is four tiles; waves beyond them fill what another wave fills, with the same
  constexpr int SC_WAVES = WL ? STILES / 4 : 1;
  static_assert(STILES % 4 == 0 && SC_WAVES <= NW, "a wave fills the scales of four tiles at most");
  const int sc_wave = __builtin_amdgcn_readfirstlane(wave % SC_WAVES);
  const uint8_t* sc_base = nullptr;
  if constexpr (WL) {
    const int t = sc_wave * 4 + (lane >> 4);
    sc_base = (t < BNT ? a.ws + (size_t)w_tile(t) * s_tile
                       : a.xs + (size_t)min(m0 / 16 + t - BNT, (a.M - 1) / 16) * s_tile) + (lane & 15) * 16;
  }
  const int n_kt = X4 ? (units + UPT - 1) / UPT : units;
  // Tile kt of K into the buffer at `at`; past the last tile the last one again, which nobody reads: the
  // loop has no branch then, over which the compiler would move matrix instructions.
  auto fill = [&](int kt, uint32_t at, int p) MM_INLINE {
    at += lds0 + (p * NW + wave) * 1024;
    const size_t k = min(kt, n_kt - 1);
    if (X4) {
      lds_fill(at, fill_base[p] + k * XT, lane16);
    } else if (p >= XF) {
      lds_fill(at, fill_base[p] + k * 1024, lane16);
    } else {                                                // (the offset made anew each time: held, it would cost a register a fill)
      int row = fill_row;
      asm volatile("" : "+v"(row));
      row = min(row + p * NW * 4, a.M - 1 - m0);
      lds_fill(at, fill_base[p] + k * 256, (uint32_t)row * (uint32_t)a.ldx * 2 + fill_piece);
    }
  };
  auto fill_scales = [&](int q) MM_INLINE {
    if constexpr (WL) {
      uint32_t m0_was;
      asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, off\n\ts_mov_b32 m0, %0"
                   : "=&s"(m0_was) : "s"(lds0 + NBUF * BUF + (q % NSB) * SB + sc_wave * 1024),
                     "v"(sc_base + (size_t)min(q, quads - 1) * 256) : "memory");
    }
  };

  f32x4 acc[NTW][MTW];
#pragma unroll
  for (int nt = 0; nt < NTW; ++nt)
#pragma unroll
    for (int mt = 0; mt < MTW; ++mt) acc[nt][mt] = f32x4{0.f, 0.f, 0.f, 0.f};

  // ---- fragments.  The matrix instructions of a step go by row tile of X: once a tile's are issued,
  // its fragment of a later step is read into the same registers.  Addresses are kept few: the compiler
  // would hold one for every read of the loop and run out of registers.
  typedef uint32_t u4_raw __attribute__((ext_vector_type(4)));
  Frag xf[AHEAD][MTW];
  Frag wf[2][X4 ? NTW : 1];
  u4_raw wc[2][X4 ? 1 : NTW];                               // W's codes of a tile of K (and, from registers, its scales)
  uint32_t wsc[2][X4 || WL ? 1 : NTW];
  constexpr int NS = X4 ? NTW + MTW : WL ? NTW : 1;         // scales of a quad: W's tiles, then X's; and of the next
  uint32_t sc[NS], sc_next[NS];
  const uint32_t x_lane = lds0 + wm * MTW * (X4 ? XT : 4096) + (X4 ? lane16 : r * 256 + ((g * 4) ^ r) * 16);
  const uint32_t w_lane = lds0 + XB + lane16;
  typedef const __attribute__((address_space(3))) u4_raw* lds_u4;
  typedef const __attribute__((address_space(3))) uint32_t* lds_u1;
  typedef const __attribute__((address_space(1))) u4_raw* global_u4;
  typedef const __attribute__((address_space(1))) uint32_t* global_u1;
  auto plus = [&](uint32_t lane_at, uint32_t by) MM_INLINE {
    uint32_t at;
    asm volatile("v_add_u32 %0, %1, %2" : "=v"(at) : "s"(by), "v"(lane_at));
    return at;
  };
  auto x_step = [&](uint32_t buf, int step) MM_INLINE {     // (piece 4 g + step of row r lies at its xor with r)
    uint32_t at = x_lane;
    if constexpr (!X4) asm volatile("v_xor_b32 %0, %1, %2" : "=v"(at) : "s"(step * 16), "v"(x_lane));
    return plus(at, buf + (X4 ? step * 1024 : 0));
  };
  auto lds_read = [&](uint32_t at) MM_INLINE {
    const u4_raw v = *(lds_u4)(uintptr_t)at;
    Frag f;
    f.u = make_uint4(v.x, v.y, v.z, v.w);
    return f;
  };
  auto read_x = [&](uint32_t at, int mt) MM_INLINE { return lds_read(at + mt * (X4 ? XT : 4096)); };
  auto read_w = [&](uint32_t at, int nt) MM_INLINE { return lds_read(at + wave_tile(nt) * XT); };
  auto read_codes = [&](uint32_t at, int nt) MM_INLINE { return *(lds_u4)(uintptr_t)(at + wave_tile(nt) * 1024); };
  auto read_scale = [&](uint32_t at, int i) MM_INLINE {
    return *(lds_u1)(uintptr_t)(at + (i < NTW ? wave_tile(i) : BNT + wm * MTW + i - NTW) * 256);
  };
  auto load_w = [&](int kt, int set) MM_INLINE {
#pragma unroll
    for (int nt = 0; nt < NTW; ++nt) {
      const size_t t = w_tile(wave_tile(nt));
      const uint8_t* codes = a.wc + t * c_tile + (size_t)kt * 1024;
      const uint8_t* scales = a.ws + t * s_tile + (size_t)(kt >> 2) * 256;
      asm volatile("" : "+s"(codes), "+s"(scales));
      wc[set][nt] = *(global_u4)(codes + lane16);
      wsc[set][nt] = *(global_u1)(scales + lane4);
    }
  };

  each<FAR>([&](auto b) MM_INLINE {
    if (b % TPQ == 0) fill_scales(b / TPQ);
    each<FILLS>([&](auto p) MM_INLINE { fill(b, b * BUF, p); });
  });
  // (the compiler is told that it has W's codes: else it would wait for them, and with them for every
  // load into LDS behind them, inside the loop)
  auto have_w = [&](int set) MM_INLINE {
#pragma unroll
    for (int nt = 0; nt < NTW; ++nt) asm volatile("" : "+v"(wc[set][nt]), "+v"(wsc[set][nt]));
  };
  if constexpr (!WL) {
    load_w(0, 0);
    have_w(0);
  }
  // What this wave asked for has arrived, but for the loads of the last `tiles` tiles; then all waves.
  auto arrived = [&](auto tiles) MM_INLINE {
    constexpr int LEFT = WL ? decltype(tiles)::value * FILLS : 0;
    if constexpr (EARLY) {
      asm volatile("s_waitcnt vmcnt(%0)" : : "n"(LEFT) : "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(LEFT) : "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    }
  };
  arrived(std::integral_constant<int, FAR - 1>{});
#pragma unroll
  for (int ahead = 0; ahead < AHEAD; ++ahead) {
    const uint32_t x_at = x_step(0, ahead);
#pragma unroll
    for (int mt = 0; mt < MTW; ++mt) xf[ahead][mt] = read_x(x_at, mt);
    if constexpr (X4) {
#pragma unroll
      for (int nt = 0; nt < NTW; ++nt) wf[ahead][nt] = read_w(w_lane + ahead * 1024, nt);
    }
  }
  if constexpr (WL) {
#pragma unroll
    for (int i = 0; i < NS; ++i) sc[i] = read_scale(lds0 + NBUF * BUF + lane4, i);
    if constexpr (!X4) {
#pragma unroll
      for (int nt = 0; nt < NTW; ++nt) wc[0][nt] = read_codes(w_lane, nt);
    }
  }

  // One tile of K, the turn-th of TURNS: it lies in the buffer at `here`, the next one in that at `there`, and
  // the one FAR tiles on goes into that at `to`.
  auto round = [&](int kt, auto turn, uint32_t here, uint32_t there, uint32_t to) MM_INLINE {
    constexpr int TURN = decltype(turn)::value, CUR = TURN & 1, NEXT = CUR ^ 1, IN_QUAD = TURN % TPQ;
    constexpr bool NEW_SCALES = WL && IN_QUAD == TPQ - 1;   // the next tile's are another quad's
    if constexpr (!WL) load_w(min(kt + 1, n_kt - 1), NEXT);
    each<STEPS>([&](auto step) MM_INLINE {
      constexpr int S = decltype(step)::value, SET = (TURN * STEPS + S) & 1;
      constexpr int XS = EARLY ? SET : 0;
      constexpr bool BORDER = S == BSTEP;                   // from here on everything read is the next tile's
      constexpr int RS = (S + AHEAD) % STEPS;               // the step whose fragments are read
      if constexpr (BORDER) {
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (!WL) have_w(NEXT);
        arrived(std::integral_constant<int, FAR - 2>{});
      }
      const uint32_t from = S >= BSTEP ? there : here;
      const uint32_t x_at = x_step(from, RS);
      uint32_t w_at = 0, s_at = 0;
      Frag w[X4 ? 1 : NTW];
      if constexpr (X4 || (WL && BORDER)) w_at = plus(w_lane, from + (X4 ? RS * 1024 : 0));
      if constexpr (NEW_SCALES && BORDER) s_at = plus(lane4, lds0 + NBUF * BUF + ((kt + 1) / TPQ % NSB) * SB);
      if constexpr (!X4) {
#pragma unroll
        for (int nt = 0; nt < NTW; ++nt) {
          const uint32_t e = WL ? sc[nt] >> (8 * IN_QUAD) : wsc[CUR][nt] >> (8 * (kt & 3));
          w[nt] = mx4_widen(wc[CUR][nt][S], mx4_scale(e & 255u));
        }
      }
      each<MTW>([&](auto mtc) MM_INLINE {
        constexpr int MT = decltype(mtc)::value;
        __builtin_amdgcn_sched_barrier(0);
        // this group's share of the loads into the buffer that is left
        if constexpr (BORDER) {
          if (MT == 0 && (TURN + FAR) % TPQ == 0) fill_scales((kt + FAR) / TPQ);
#pragma unroll
          for (int p = FILLS * MT / MTW; p < FILLS * (MT + 1) / MTW; ++p) fill(kt + FAR, to, p);
        }
        each<NTW>([&](auto ntc) MM_INLINE {
          constexpr int NT = decltype(ntc)::value;
          if constexpr (X4)
            acc[NT][MT] = mx4_mfma<IN_QUAD * UPT + S, IN_QUAD * UPT + S>(wf[SET][NT].u, sc[NT], xf[XS][MT].u, sc[NTW + MT], acc[NT][MT]);
          else
            acc[NT][MT] = mfma_bf16(w[NT], xf[XS][MT], acc[NT][MT]);
        });
        __builtin_amdgcn_sched_barrier(0);
        // its share of the reads, behind them
        xf[XS][MT] = read_x(x_at, MT);
        if constexpr (X4) {
          if constexpr (!EARLY) {
#pragma unroll
            for (int nt = NTW * MT / MTW; nt < NTW * (MT + 1) / MTW; ++nt) wf[SET ^ 1][nt] = read_w(w_at, nt);
          } else if constexpr (MT == MTW - 1) {              // (this step's are done with)
#pragma unroll
            for (int nt = 0; nt < NTW; ++nt) wf[SET][nt] = read_w(w_at, nt);
          }
        } else if constexpr (WL && BORDER) {
#pragma unroll
          for (int nt = NTW * MT / MTW; nt < NTW * (MT + 1) / MTW; ++nt) wc[NEXT][nt] = read_codes(w_at, nt);
        }
        if constexpr (NEW_SCALES && BORDER) {
#pragma unroll
          for (int i = NS * MT / MTW; i < NS * (MT + 1) / MTW; ++i) sc_next[i] = read_scale(s_at, i);
        }
      });
    });
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (NEW_SCALES) {
#pragma unroll
      for (int i = 0; i < NS; ++i) sc[i] = sc_next[i];
    }
  };
  // where tile kt + FAR goes: FAR is the number of buffers, or one less
  uint32_t here = 0, there = NBUF > 1 ? BUF : 0, to = FAR % NBUF * BUF;
  auto turn_over = [&](int kt, auto turn) MM_INLINE {
    round(kt, turn, here, there, to);
    here = there;
    there = there == (NBUF - 1) * BUF ? 0 : there + BUF;
    to = to == (NBUF - 1) * BUF ? 0 : to + BUF;
  };
  int kt = 0;
  for (; kt + TURNS <= n_kt; kt += TURNS) each<TURNS>([&](auto turn) MM_INLINE { turn_over(kt + turn, turn); });
  each<TURNS - 1>([&](auto turn) MM_INLINE {
    if (kt + turn < n_kt) turn_over(kt + turn, turn);
  });
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");       // the last loads into LDS have landed too

  // ---- epilogue: lane holds C[m = .. + r][n = .. + 4 g + e]
  constexpr int OUT_NT = GATED ? NTW / 2 : NTW;
  const int n_wave = (nt_blk * (GATED ? BNT / 2 : BNT) + wn * OUT_NT) * 16, m_wave = m0 + wm * MTW * 16;
  float bias[OUT_NT][4];
#pragma unroll
  for (int nt = 0; nt < OUT_NT; ++nt)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int n = n_wave + nt * 16 + 4 * g + e;
      bias[nt][e] = !GATED && a.bias != nullptr && n < a.n_out ? a.bias[n] : 0.f;
    }
  auto value = [&](int nt, int mt, float (&v)[4]) MM_INLINE {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = acc[nt][mt][e];
      if (GATED) {
        v[e] = mx4_gated<sizeof(OutT) == 4>(a.act, acc[nt][mt][e], acc[nt + NTW / 2 < NTW ? nt + NTW / 2 : nt][mt][e]);
      } else {
        v[e] += bias[nt][e];
      }
    }
  };
  // Each wave turns its tile round through a region of LDS of its own, 16 rows of X at a time, rows 16
  // bytes longer than they are so that the 16 rows of a write fall into different banks, and then stores
  // whole rows: 16 bytes a lane, or where rows of C do not begin at multiples of that an element a lane,
  // neighbours in neighbouring lanes (3,000 rows, K 64, in float32, us: 28,000 outputs 97 and straight from
  // the sums, 64 bytes of a row at a time, 148; 28,001 outputs 118 and 249; in bfloat16 28,001 92, by eight
  // neighbours a lane 192).
  __syncthreads();                                          // every wave has read the last tile
  constexpr int ES = sizeof(OutT), COLS = OUT_NT * 16, ROW_B = COLS * ES + 16, VEC = 16 / ES;
  constexpr int LPR = COLS / VEC, RPP = 64 / LPR;           // lanes a row, rows a store
  unsigned char* mine = lds + wave * (16 * ROW_B);
  const bool whole = a.n_out % VEC == 0;
#pragma unroll
  for (int mt = 0; mt < MTW; ++mt) {
#pragma unroll
    for (int nt = 0; nt < OUT_NT; ++nt) {
      float v[4];
      value(nt, mt, v);
      unsigned char* dst = mine + r * ROW_B + (nt * 16 + 4 * g) * ES;
      if constexpr (ES == 4) *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
      else *reinterpret_cast<uint2*>(dst) = make_uint2(pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3]));
    }
    // (a wave's accesses to LDS run in order; the compiler may not move one lane's read over another's write)
    asm volatile("" ::: "memory");
    const int m_tile = m_wave + mt * 16;
    if (whole) {
      const int n = n_wave + lane % LPR * VEC;
#pragma unroll
      for (int pass = 0; pass < (16 + RPP - 1) / RPP; ++pass) {
        const int row = pass * RPP + lane / LPR;
        if (row < 16 && m_tile + row < a.M && n < a.n_out)
          *reinterpret_cast<uint4*>((OutT*)a.C + (size_t)(m_tile + row) * a.n_out + n) =
              *reinterpret_cast<const uint4*>(mine + row * ROW_B + lane % LPR * 16);
      }
    } else {
      const int n = n_wave + lane % COLS;
#pragma unroll
      for (int row0 = 0; row0 < 16; row0 += 64 / COLS) {
        const int row = row0 + lane / COLS;
        if (m_tile + row < a.M && n < a.n_out)
          ((OutT*)a.C)[(size_t)(m_tile + row) * a.n_out + n] = reinterpret_cast<const OutT*>(mine + row * ROW_B)[lane % COLS];
      }
    }
    asm volatile("" ::: "memory");
  }
}

template <bool X4, int NBUF, bool EARLY, int WM, int WN, int MTW, int NTW, int EPI, typename OutT>
static int launch_mx4_many(Mx4ManyArgs a) {
  typedef ManyShape<X4, NBUF, EARLY, WM, WN, MTW, NTW> Shape;
  constexpr int BM = Shape::BM, BNT = Shape::BNT, NW = WM * WN;
  constexpr int OUT_NT = EPI == MM_EPI_GATED ? NTW / 2 : NTW;
  constexpr int TURN = NW * 16 * (OUT_NT * 16 * (int)sizeof(OutT) + 16);
  constexpr int LDS_BYTES = Shape::BYTES > TURN ? Shape::BYTES : TURN;
  static_assert(LDS_BYTES <= 160 * 1024, "shared memory of a unit");
  const int out_tiles = (a.n_out + 15) / 16, per = EPI == MM_EPI_GATED ? BNT / 2 : BNT;
  a.m_tiles = (a.M + BM - 1) / BM;
  a.n_tiles = (out_tiles + per - 1) / per;
  // Surplus blocks, where tiles of W are no multiple of 8, leave at once, but each has to be given its LDS first:
  // none along X's rows (with bands of 8 always full, 64 rows, K 14,336 in seven slices, 4,096 outputs: 19.0 us against 16.5).
  const long long blocks = 8LL * a.m_tiles * ((a.n_tiles + 7) / 8);
  if (blocks > 0x7fffffffLL) return LLM_ERR_ARG;
  // more than 64 KiB of LDS has to be asked for, once per device and kernel
  static bool asked[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return LLM_ERR_LAUNCH;
  if (!asked[dev]) {
    if (hipFuncSetAttribute((const void*)gemm_mx4_many_kernel<X4, NBUF, EARLY, WM, WN, MTW, NTW, EPI, OutT>,
                            hipFuncAttributeMaxDynamicSharedMemorySize, LDS_BYTES) != hipSuccess)
      return LLM_ERR_LAUNCH;
    asked[dev] = true;
  }
  const dim3 grid((unsigned)blocks, (a.quads + a.slice_quads - 1) / a.slice_quads);
  gemm_mx4_many_kernel<X4, NBUF, EARLY, WM, WN, MTW, NTW, EPI, OutT><<<grid, NW * 64, LDS_BYTES, a.stream>>>(a);
  return llm_launch_status();
}

// Forms: rows of X by rows of W a block.  0, 256 x 256: fewest bytes a product, one block a unit.  1,
// 128 x 128 (MXFP4) or 128 x 256 (bfloat16, where three tiles of K fit): more blocks, for products that
// would leave units idle in the last round (bfloat16, 4,096 rows, K 4,096, 6,144 outputs: 157 us against
// 167).  2, 64 x 128: several blocks a unit, which cover each other's waits.  3, 64 x 128 with four tiles of
// K held and fragments two steps ahead: for a block a unit or less, where a block waits for memory (1.5 us
// from a weight that no cache holds).  In bfloat16 that form has eight waves (128 rows, K 4,096, 6,144
// outputs, us: 19.6, by four waves 22.3, form 2 22.9).  4, 64 x 64, for products that even so give a block to a
// fraction of the units (128 rows, us by form 3 and 4: K 2,048, 2,048 outputs in bfloat16 10.8 and 9.5, in MXFP4 6.6
// and 5.8, K 4,096, 6,144 outputs in MXFP4 10.1 and 8.2); in MXFP4 it holds six tiles of K (four: 8.8).
// Left as they are, measured: four tiles of 128 elements instead of two of 256 in form 0 of MXFP4 (61.2 us
// against 59.6 at 4,096 rows, K 4,096, 6,144 outputs), and the widening taken out of form 0 in bfloat16
// (no change): neither latency nor the vector units bound the large products.
#define MM_FORMS 5
template <bool X4, int EPI, typename OutT>
static int pick_mx4_many(const Mx4ManyArgs& a, int form) {
  if constexpr (X4) {
    switch (form) {
      case 0: return launch_mx4_many<true, 2, false, 2, 4, 8, 4, EPI, OutT>(a);
      case 1: return launch_mx4_many<true, 2, false, 2, 2, 4, 4, EPI, OutT>(a);
      case 2: return launch_mx4_many<true, 2, false, 1, 4, 4, 2, EPI, OutT>(a);
      case 3: return launch_mx4_many<true, 4, true, 1, 4, 4, 2, EPI, OutT>(a);
      case 4: return launch_mx4_many<true, 6, true, 2, 2, 2, 2, EPI, OutT>(a);
    }
  } else {
    switch (form) {
      case 0: return launch_mx4_many<false, 2, false, 2, 4, 8, 4, EPI, OutT>(a);
      case 1: return launch_mx4_many<false, 3, false, 2, 4, 4, 4, EPI, OutT>(a);
      case 2: return launch_mx4_many<false, 2, false, 1, 4, 4, 2, EPI, OutT>(a);
      case 3: return launch_mx4_many<false, 4, true, 2, 4, 2, 2, EPI, OutT>(a);
      case 4: return launch_mx4_many<false, 4, true, 2, 2, 2, 2, EPI, OutT>(a);
    }
  }
  return LLM_ERR_ARG;
}

template <bool X4>
static int mx4_many(const Mx4ManyArgs& a, int epilogue, int out_dtype, int form) {
  if (epilogue == MM_EPI_GATED) return out_dtype == LLM_DTYPE_BF16 ? pick_mx4_many<X4, MM_EPI_GATED, bf16_t>(a, form) : LLM_ERR_ARG;
  if (out_dtype == LLM_DTYPE_BF16) return pick_mx4_many<X4, MM_EPI_NONE, bf16_t>(a, form);
  if (out_dtype == LLM_DTYPE_F32) return pick_mx4_many<X4, MM_EPI_NONE, float>(a, form);
  return LLM_ERR_ARG;
}

// W [N, K] as mx4.h lays it out.  X: bfloat16 rows ldx apart with xs null (their length K and ldx
// multiples of 128, what lies beyond W's width zero), or codes with their scales in xs.  epilogue 0:
// C [M, N] of out_dtype, plus bias[n] if not null; 1 | act << 4: C [M, N / 2] in bfloat16, the gate
// through an activation of common.h, N / 2 a multiple of 16.  form: 0 .. 4, see above.  With k_split
// above 1 (epilogue 0, float32, no bias) C is [k_split, M, N], the products over as many slices of K of
// ceil(quads / k_split) quads of 512 elements; every slice has elements.
extern "C" int llm_gemm_mx4_many(const void* X, const void* xs, int ldx, const void* wc, const void* ws,
                                 const float* bias, void* C, int epilogue, int out_dtype, int M, int N, int K,
                                 int form, int k_split, hipStream_t stream) {
  if (M <= 0) return LLM_OK;
  const int act = epilogue >> 4;
  epilogue &= 15;
  if (epilogue != MM_EPI_NONE && epilogue != MM_EPI_GATED) return LLM_ERR_ARG;
  if (N <= 0 || K <= 0 || act < 0 || act >= LLM_ACT_COUNT || (epilogue != MM_EPI_GATED && act != 0)) return LLM_ERR_ARG;
  if (X == nullptr || wc == nullptr || ws == nullptr || C == nullptr) return LLM_ERR_ARG;
  if ((((uintptr_t)X) | ((uintptr_t)wc) | ((uintptr_t)ws) | ((uintptr_t)C) | ((uintptr_t)xs)) & 15) return LLM_ERR_ARG;
  if (xs == nullptr && (ldx < K || (ldx & 127) || (K & 127) || ldx > (1 << 22))) return LLM_ERR_ARG;   // (offsets within a block's rows stay below 2^32)
  if (epilogue == MM_EPI_GATED && ((N & 31) || bias != nullptr)) return LLM_ERR_ARG;
  Mx4ManyArgs a{};
  a.X = (const bf16_t*)X;
  a.xc = (const uint8_t*)X;
  a.xs = (const uint8_t*)xs;
  a.wc = (const uint8_t*)wc;
  a.ws = (const uint8_t*)ws;
  a.bias = bias;
  a.C = C;
  a.M = M;
  a.N = N;
  a.n_out = epilogue == MM_EPI_GATED ? N / 2 : N;
  a.ldx = ldx;
  a.units = mx4_units(K);
  a.quads = mx4_quads(K);
  a.act = act;
  a.stream = stream;
  if (k_split < 1 || form < 0 || form >= MM_FORMS) return LLM_ERR_ARG;
  a.slice_quads = (a.quads + k_split - 1) / k_split;
  if (k_split > 1 && (epilogue != MM_EPI_NONE || out_dtype != LLM_DTYPE_F32 || bias != nullptr ||
                      (a.quads + a.slice_quads - 1) / a.slice_quads != k_split))
    return LLM_ERR_ARG;
  return xs == nullptr ? mx4_many<false>(a, epilogue, out_dtype, form) : mx4_many<true>(a, epilogue, out_dtype, form);
}

// The slices' sums parts [n_parts, M, N] (or one product whose gate and up lie in no whole tiles), added
// in their order, plus bias or through the gate, to C of out_dtype: four columns a thread (N and n_out multiples of 4), or one.
template <int VEC, bool GATED, typename OutT>
__global__ __launch_bounds__(256) void mx4_join_kernel(const float* __restrict__ parts, int n_parts, const float* bias,
                                                       OutT* __restrict__ C, size_t M, int N, int n_out, int act) {
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  const int per_row = n_out / VEC;
  const size_t m = i / per_row;
  const int n = (int)(i - m * per_row) * VEC;
  if (m >= M) return;
  float v[VEC], u[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) v[e] = u[e] = 0.f;
  for (int p = 0; p < n_parts; ++p) {
    const float* src = parts + ((size_t)p * M + m) * N + n;
    if constexpr (VEC == 4) {
      const float4 q = *reinterpret_cast<const float4*>(src);
      v[0] += q.x; v[1] += q.y; v[2] += q.z; v[3] += q.w;
      if (GATED) {
        const float4 w = *reinterpret_cast<const float4*>(src + n_out);
        u[0] += w.x; u[1] += w.y; u[2] += w.z; u[3] += w.w;
      }
    } else {
      v[0] += src[0];
      if (GATED) u[0] += src[n_out];
    }
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    if (GATED) v[e] = mx4_gated<sizeof(OutT) == 4>(act, v[e], u[e]);
    else if (bias != nullptr) v[e] += bias[n + e];
  }
  OutT* dst = C + m * n_out + n;
  if constexpr (VEC == 4) Conv4<OutT>::store(dst, make_float4(v[0], v[1], v[2], v[3]));
  else Conv<OutT>::store(dst, v[0]);
}

extern "C" int llm_mx4_join(const void* parts, int n_parts, const float* bias, void* C, int epilogue, int out_dtype,
                            int M, int N, hipStream_t stream) {
  if (M <= 0) return LLM_OK;
  const int act = epilogue >> 4;
  const bool gated = (epilogue & 15) == MM_EPI_GATED;
  if (N <= 0 || n_parts <= 0 || act < 0 || act >= LLM_ACT_COUNT || parts == nullptr || C == nullptr || (gated && (N & 1))) return LLM_ERR_ARG;
  const int n_out = gated ? N / 2 : N, vec = (n_out & 3) ? 1 : 4;
  const size_t blocks = ((size_t)M * (n_out / vec) + 255) / 256;
  if (blocks > 0x7fffffff) return LLM_ERR_ARG;
#define MX4_JOIN(V, G, T) \
  mx4_join_kernel<V, G, T><<<(unsigned)blocks, 256, 0, stream>>>((const float*)parts, n_parts, bias, (T*)C, M, N, n_out, act)
#define MX4_JOIN_T(T)                                                 \
  if (gated) { if (vec == 4) MX4_JOIN(4, true, T); else MX4_JOIN(1, true, T); } \
  else { if (vec == 4) MX4_JOIN(4, false, T); else MX4_JOIN(1, false, T); }
  if (out_dtype == LLM_DTYPE_BF16) { MX4_JOIN_T(bf16_t) }
  else if (out_dtype == LLM_DTYPE_F32) { MX4_JOIN_T(float) }
  else return LLM_ERR_ARG;
#undef MX4_JOIN_T
#undef MX4_JOIN
  return llm_launch_status();
}
