// What the products for few rows do with their sums beside storing them: rotate them and write them to
// the cache, or add them into the residual stream and prepare the norm that reads it next.  A thread
// finishes four neighbouring columns n .. n + 3 of a row m.
#pragma once
#include "mfma.h"

// Rotary epilogue of a stacked q|k|v projection whose rotating pairs lie side by side (pair j of a head
// at 2j, 2j+1).  Head sizes are multiples of 16, so that four columns belong to one head.
struct RowRope {
  const float* bias;       // [outputs of the projection] or null
  const float* cos_t;      // [positions, rot_dim / 2]
  const float* sin_t;
  const int* tok_pos;      // [M] position of each row's token
  const int* tok_seq;      // [M] its sequence in the step
  const int* seq_slot;     // [sequences] slot of each sequence
  const int* table;        // [slots, table_stride] page of (slot, position / 64)
  bf16_t* k_pages;
  bf16_t* v_pages;
  int table_stride, n_heads, n_kv, hd, rot_dim, write_kv;
};

// What the rotary epilogue of RT tiles of outputs (16 columns apart, from column n0 on) needs from memory
// beside the sums, asked for before they are there.
template <int RT>
struct RopeAhead {
  int pos, page;
  float2 cos[RT], sin[RT];

  __device__ __forceinline__ void load(const RowRope& rope, int m, int n0) {
    pos = rope.tok_pos[m];
    page = 0;
    const int q_dim = rope.n_heads * rope.hd, kv_dim = rope.n_kv * rope.hd;
#pragma unroll
    for (int ort = 0; ort < RT; ++ort) {
      const int n = n0 + ort * 16, d = n % rope.hd;
      cos[ort] = make_float2(1.f, 1.f);
      sin[ort] = make_float2(0.f, 0.f);
      if (n < q_dim + kv_dim && d < rope.rot_dim) {       // rot_dim is even; d is a multiple of 4
        const float* cr = rope.cos_t + (size_t)pos * (rope.rot_dim / 2) + (d >> 1);
        const float* sr = rope.sin_t + (size_t)pos * (rope.rot_dim / 2) + (d >> 1);
        cos[ort].x = cr[0];
        sin[ort].x = sr[0];
        if (d + 2 < rope.rot_dim) {
          cos[ort].y = cr[1];
          sin[ort].y = sr[1];
        }
      }
    }
    if (rope.write_kv && n0 + (RT - 1) * 16 >= q_dim) {
      const int slot = rope.seq_slot[rope.tok_seq[m]];
      page = rope.table[(size_t)slot * rope.table_stride + pos / 64];
    }
  }
};

// The same in three steps without a branch, for a kernel whose registers a branch between its first loads
// and its loop would double: what the first step asks for has to be there for the second, and so on; the
// first goes in front of the kernel's own loads, which then need not arrive before the second.  m is a row
// that exists.
template <int RT>
struct RopeSteps : RopeAhead<RT> {
  int seq, slot;

  __device__ __forceinline__ void first(const RowRope& rope, int m) {
    this->pos = rope.tok_pos[m];
    seq = (rope.write_kv ? rope.tok_seq : rope.tok_pos)[m];
  }
  __device__ __forceinline__ void second(const RowRope& rope, int n0) {
    const int half = rope.rot_dim / 2, qk = (rope.n_heads + rope.n_kv) * rope.hd;
    const float* ct = half ? rope.cos_t : (const float*)rope.tok_pos;       // (somewhere that can be read)
    const float* st = half ? rope.sin_t : (const float*)rope.tok_pos;
#pragma unroll
    for (int ort = 0; ort < RT; ++ort) {
      const int n = n0 + ort * 16, d = n % rope.hd;
      const bool x = n < qk && d < rope.rot_dim, y = n < qk && d + 2 < rope.rot_dim;
      const size_t at = (size_t)this->pos * half + (d >> 1);
      const float c0 = ct[x ? at : 0], c1 = ct[y ? at + 1 : 0], s0 = st[x ? at : 0], s1 = st[y ? at + 1 : 0];
      this->cos[ort] = make_float2(x ? c0 : 1.f, y ? c1 : 1.f);
      this->sin[ort] = make_float2(x ? s0 : 0.f, y ? s1 : 0.f);
    }
    slot = (rope.write_kv ? rope.seq_slot : rope.tok_pos)[rope.write_kv ? seq : 0];
  }
  __device__ __forceinline__ void third(const RowRope& rope) {
    const size_t at = (size_t)slot * rope.table_stride + this->pos / 64;
    this->page = (rope.write_kv ? rope.table : rope.tok_pos)[rope.write_kv ? at : 0];
  }
};

// Bias, rotation, and the store: q to q_out [M, n_heads * hd], k and v to their place in the cache.
template <int RT>
__device__ __forceinline__ void rope_store(const RowRope& rope, const RopeAhead<RT>& ahead, int ort, float (&v)[4],
                                           int m, int n, bf16_t* q_out) {
  if (rope.bias) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += rope.bias[n + e];
  }
  const int q_dim = rope.n_heads * rope.hd, kv_dim = rope.n_kv * rope.hd;
  const int pos = ahead.pos;
  const int d = n % rope.hd;
  {                                               // q and k rotate; elsewhere the angle is zero
    const float c0 = ahead.cos[ort].x, s0 = ahead.sin[ort].x, c1 = ahead.cos[ort].y, s1 = ahead.sin[ort].y;
    const float a0 = v[0], a1 = v[1], a2 = v[2], a3 = v[3];
    v[0] = a0 * c0 - a1 * s0;
    v[1] = a1 * c0 + a0 * s0;
    v[2] = a2 * c1 - a3 * s1;
    v[3] = a3 * c1 + a2 * s1;
  }
  uint2 pk;
  pk.x = pack2_bf16(v[0], v[1]);
  pk.y = pack2_bf16(v[2], v[3]);
  if (n < q_dim) {
    *reinterpret_cast<uint2*>(q_out + (size_t)m * q_dim + n) = pk;
  } else if (rope.write_kv) {
    const int page = ahead.page;
    const int kn = n - q_dim;
    if (kn < kv_dim) {
      const int kvh = kn / rope.hd;
      *reinterpret_cast<uint2*>(rope.k_pages + ((size_t)page * rope.n_kv + kvh) * llm_key_block(rope.hd) +
                                llm_key_offset(pos % 64, d)) = pk;
    } else {
      const int kvh = (kn - kv_dim) / rope.hd;
      bf16_t* vp = rope.v_pages + ((size_t)page * rope.n_kv + kvh) * llm_value_block(rope.hd) +
                   llm_value_offset(rope.hd, d, pos % 64);         // dims d .. d + 3 lie 32 apart
      vp[0] = (bf16_t)(pk.x & 0xffffu);
      vp[32] = (bf16_t)(pk.x >> 16);
      vp[64] = (bf16_t)(pk.y & 0xffffu);
      vp[96] = (bf16_t)(pk.y >> 16);
    }
  }
}

// The sums added into the stream C [M, ldc] (prev: what it holds), the new stream times the next norm's
// weight nw to raw, rounded, and the sums of squares of its tiles of 16 columns to ssq_out.  ldc is a
// multiple of 16: a tile is whole or absent.  Every lane of the wave comes along; lanes 16 apart (g = lane
// / 16) hold the columns of a tile of the same row, and `on` says whether this lane's exist.
__device__ __forceinline__ void norm_store(bool on, float (&v)[4], const float (&prev)[4], const float (&nw)[4], int m,
                                           int n, int ldc, int g, float* C, bf16_t* raw, float* ssq_out) {
  float ss = 0.f;
  if (on) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] += prev[e];
      ss += v[e] * v[e];
    }
    *reinterpret_cast<float4*>(C + (size_t)m * ldc + n) = make_float4(v[0], v[1], v[2], v[3]);
    uint2 pk;
    pk.x = pack2_bf16(v[0] * nw[0], v[1] * nw[1]);
    pk.y = pack2_bf16(v[2] * nw[2], v[3] * nw[3]);
    *reinterpret_cast<uint2*>(raw + (size_t)m * ldc + n) = pk;
  }
  ss += __shfl_xor(ss, 16, 64);
  ss += __shfl_xor(ss, 32, 64);
  if (on && g == 0) ssq_out[(size_t)m * (ldc / 16) + n / 16] = ss;
}
