// One wave's share of a decode: the steps of one (sequence, kv head) streamed through the
// matrix cores, and what goes with it (the span a query sees, the running state, the final
// factor). The arithmetic and the operand arrangement are described in kept_decode.hip; used
// there and, for the tokens behind a shared prefix, in shared_decode.hip.
#pragma once

#include "kept.hpp"

namespace gkv {

constexpr int kKeptAux = 2;            // nontemporal: each K/V byte is read once
constexpr int kHeads = 8;              // query heads per kv head, at most
constexpr int kPieceFloats = kHeads * kHeadDim;
constexpr int kPieceMl = 2 * kHeads;   // (m, l) of a piece's heads
constexpr float kLowest = -1e30f;      // the running maximum before any score (log2 units)

struct KeptDecodeArgs {
  const float *q;
  int64_t q_stride;
  const float *cos_tab, *sin_tab;
  const int32_t *seq_lens;
  const char *kc, *vc;
  const float *scales;
  const int32_t *table;
  int table_stride, num_blocks;
  KeptRow row;
  int window, max_len;
  const float *sinks; // NULL: none
  int B, G, n_kv_heads;
  int parts, heads_per_wg; // whole: waves per (sequence, head), heads per workgroup
  int max_ranges;          // ranges: waves launched per kv head
  int4 *cuts;              // ranges: {sequence, its first step, its end, T} of the sequence that range
                           // r starts inside of (sequence -1: at a sequence's start, or no range)
  float *ws_ml, *ws_o;     // [range][2][n_kv_heads]: a range's first and last piece
  void *out;
  int64_t out_stride;
  int out_bf16;
  uint32_t *dev_err;
};

// What a sequence's query sees: blocks 0 .. first_blocks - 1, then from
// logical block win0 on, n_blocks in all.
struct Span {
  int L, first_blocks, win0, n_blocks;
  int ring0; // win0's place in the ring
};

__device__ __forceinline__ int span_len(const KeptDecodeArgs &a, int b) {
  return max(min(a.seq_lens[b], a.max_len), 0);
}

__device__ __forceinline__ Span span_of(const KeptDecodeArgs &a, int L) {
  Span s;
  s.L = L;
  const int nb = (L + kBlockTokens - 1) / kBlockTokens;
  if (a.window == 0) {
    s.first_blocks = s.n_blocks = nb;
    s.win0 = s.ring0 = 0;
    return s;
  }
  s.first_blocks = min(a.row.kept_blocks, nb);
  s.win0 = max(max(L - a.window, 0) / kBlockTokens, a.row.kept_blocks);
  s.n_blocks = s.first_blocks + max(nb - s.win0, 0);
  s.ring0 = a.row.ring_blocks
                ? (int)((uint32_t)(s.win0 - a.row.kept_blocks) % (uint32_t)a.row.ring_blocks)
                : 0;
  return s;
}

__device__ __forceinline__ int span_steps(const Span &s) { return (s.n_blocks + 1) / 2; }

// Table entry of the span's i-th block (a window spans at most the ring).
__device__ __forceinline__ int span_entry(const KeptDecodeArgs &a, const Span &s, int i) {
  if (i < s.first_blocks)
    return i;
  const int w = i - s.first_blocks;
  if (a.row.ring_blocks == 0)
    return s.win0 + w;
  const int e = s.ring0 + w;
  return a.row.kept_blocks + (e >= a.row.ring_blocks ? e - a.row.ring_blocks : e);
}

__device__ __forceinline__ void put(void *out, int64_t i, f32x4 v, int bf16) {
  if (bf16)
    *(u32x2 *)((uint16_t *)out + i) =
        u32x2{f32x2_to_bf16_rne(v[0], v[1]), f32x2_to_bf16_rne(v[2], v[3])};
  else
    *(f32x4 *)((float *)out + i) = v;
}

// The running state of one wave: maximum (log2 units) and weight sum of this
// lane's column, its part of O^T.
struct State {
  float m, l;
  f32x4 o[4];
};

template <bool BLK>
struct StepData {
  u32x4 k[BLK ? 2 : 4], v[BLK ? 2 : 4];
  f32x2 sc[2];   // per block: K scale, V scale (wave-uniform)
  uint32_t miss; // bit j: block j is not there (padding, or an id outside the pool)
};
constexpr int kNoBlock = -1; // the id of a step's missing second block

typedef const __attribute__((address_space(4))) int32_t *ScalarI32;
typedef const __attribute__((address_space(4))) f32x2 *ScalarF2;

// Steps s0 .. s1 - 1 of sequence b for kv head g, by one wave. R: steps of data in
// registers. FINE: three bf16 pieces where two would do for a bf16 output.
template <bool BLK, int R, bool FINE>
__device__ __forceinline__ State attend(const KeptDecodeArgs &a, int b, int g, const Span &sp,
                                        int s0, int s1) {
  constexpr int D = kHeadDim;
  constexpr int kHeadBytes = kBlockTokens * D * (BLK ? 1 : 2);
  const int lane = threadIdx.x & 63, col = lane & 15, kg = lane >> 4;
  const bool low = col >= 8;
  const int head = col & 7;
  const bool head_ok = head < a.G;
  const uint32_t k_off = lane * 16;
  const uint32_t v_off = BLK ? (col * 4 + kg) * 16 : lane * 16;

  // The query's rows and angles: dims 8kg .. +7 and 32+8kg .. +7 of the column's
  // head. Their loads go out first, as their address depends on nothing else.
  f32x4 qr[4], an[4];
  {
    const f32x4 *qp =
        (const f32x4 *)(a.q + (int64_t)b * a.q_stride + (g * a.G + (head_ok ? head : 0)) * D + 8 * kg);
    qr[0] = qp[0];
    qr[1] = qp[1];
    qr[2] = qp[8];
    qr[3] = qp[9];
    if (a.cos_tab) {
      const f32x4 *cp = (const f32x4 *)(a.cos_tab + (int64_t)(sp.L - 1) * (D / 2) + 8 * kg);
      const f32x4 *np = (const f32x4 *)(a.sin_tab + (int64_t)(sp.L - 1) * (D / 2) + 8 * kg);
      an[0] = cp[0];
      an[1] = cp[1];
      an[2] = np[0];
      an[3] = np[1];
    }
  }

  // The block ids of a step, read through the scalar cache a step before they are
  // used.
  const ScalarI32 trow = (ScalarI32)a.table + (int64_t)b * a.table_stride;
  bool bad = false;
  auto ids_of = [&](int s) -> int2 {
    int2 r{kNoBlock, kNoBlock};
    if (s < s1) {
      r.x = trow[span_entry(a, sp, 2 * s)];
      if (2 * s + 1 < sp.n_blocks)
        r.y = trow[span_entry(a, sp, 2 * s + 1)];
    }
    return r;
  };
  const char *k_head = a.kc + g * kHeadBytes, *v_head = a.vc + g * kHeadBytes;
  const char *s_head = (const char *)a.scales + g * 8;
  const uint32_t stride = (uint32_t)a.n_kv_heads * kHeadBytes; // bytes of a block
  auto load = [&](StepData<BLK> &x, int2 ids, int s) {
    x.miss = 0;
    const bool first = s < s1, second = first && 2 * s + 1 < sp.n_blocks; // which there are
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const int id = uniform(j ? ids.y : ids.x);
      const bool ok = (uint32_t)id < (uint32_t)a.num_blocks;
      bad |= !ok && (j ? second : first);
      x.miss |= ok ? 0u : 1u << j;
      const uint64_t off = (uint64_t)(ok ? (uint32_t)id : 0u) * stride;
      // a missing block reads nothing: its resource covers 0 bytes
      const __amdgpu_buffer_rsrc_t kr = head_rsrc(k_head + off, ok ? kHeadBytes : 0);
      const __amdgpu_buffer_rsrc_t vr = head_rsrc(v_head + off, ok ? kHeadBytes : 0);
      if (BLK) {
        x.sc[j] = *(ScalarF2)(s_head + off / 128);
        x.k[j] = __builtin_amdgcn_raw_buffer_load_b128(kr, k_off, 0, kKeptAux);
        x.v[j] = __builtin_amdgcn_raw_buffer_load_b128(vr, v_off, 0, kKeptAux);
      } else {
#pragma unroll
        for (int h = 0; h < 2; h++) {
          x.k[2 * j + h] = __builtin_amdgcn_raw_buffer_load_b128(kr, k_off + h * 1024, 0, kKeptAux);
          x.v[2 * j + h] = __builtin_amdgcn_raw_buffer_load_b128(vr, v_off + h * 1024, 0, kKeptAux);
        }
      }
    }
  };

  const int last_step = (sp.n_blocks - 1) / 2, win_step = a.window > 0 ? sp.first_blocks / 2 : -1;
  StepData<BLK> buf[R];
  int2 ids = ids_of(s0);
#pragma unroll
  for (int i = 0; i < R - 1; i++) {
    const int2 next = ids_of(s0 + i + 1);
    load(buf[i], ids, s0 + i);
    ids = next;
  }

  // The query, rotated at the sequence's last position, scaled, in two pieces.
  float qa[8], qb[8];
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const float y1 = qr[i / 4][i % 4], y2 = qr[2 + i / 4][i % 4];
    qa[i] = y1;
    qb[i] = y2;
    if (a.cos_tab) {
      qa[i] = rope_first(y1, y2, an[i / 4][i % 4], an[2 + i / 4][i % 4]);
      qb[i] = rope_second(y1, y2, an[i / 4][i % 4], an[2 + i / 4][i % 4]);
    }
  }
  float qf = 0.125f * kLog2e; // 1 / sqrt(64); exp -> exp2
  if (BLK) {
    // q * 2^-e has its largest element in [1, 2)
    float mx = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++)
      mx = fmaxf(mx, fmaxf(fabsf(qa[i]), fabsf(qb[i])));
    mx = fmaxf(mx, __shfl_xor(mx, 16));
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    const int e = min(max((int)(__float_as_uint(mx) >> 23), 27), 227);
    const float down = __uint_as_float((uint32_t)(254 - e) << 23);
    qf *= __uint_as_float((uint32_t)e << 23);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      qa[i] *= down;
      qb[i] *= down;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      qa[i] *= qf;
      qb[i] *= qf;
    }
  }
  u32x4 q0, q1, q2, q3; // (q2, q3: the third pieces, bf16 K and FINE)
  {
    typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
    if (BLK) {
      f16x8 x, y;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const _Float16 hx = (_Float16)qa[i], hy = (_Float16)qb[i];
        x[i] = low ? (_Float16)(qa[i] - (float)hx) : hx;
        y[i] = low ? (_Float16)(qb[i] - (float)hy) : hy;
      }
      q0 = __builtin_bit_cast(u32x4, x);
      q1 = __builtin_bit_cast(u32x4, y);
    } else {
      bf16x8_t x, y;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const __bf16 hx = (__bf16)qa[i], hy = (__bf16)qb[i];
        x[i] = low ? (__bf16)(qa[i] - (float)hx) : hx;
        y[i] = low ? (__bf16)(qb[i] - (float)hy) : hy;
      }
      q0 = __builtin_bit_cast(u32x4, x);
      q1 = __builtin_bit_cast(u32x4, y);
      if (FINE) {
        auto third = [&](float f) {
          const __bf16 h = (__bf16)f;
          const float r = f - (float)h;
          const __bf16 m = (__bf16)r;
          return low ? (__bf16)0.0f : (__bf16)(r - (float)m);
        };
#pragma unroll
        for (int i = 0; i < 8; i++) {
          x[i] = third(qa[i]);
          y[i] = third(qb[i]);
        }
        q2 = __builtin_bit_cast(u32x4, x);
        q3 = __builtin_bit_cast(u32x4, y);
      }
    }
    if (!head_ok)
      q0 = q1 = q2 = q3 = u32x4{0, 0, 0, 0};
  }

  State st;
  st.m = kLowest;
  st.l = 0.0f;
#pragma unroll
  for (int nn = 0; nn < 4; nn++)
    st.o[nn] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  // One step. After the scores' matrix ops a column's two halves hold what q's
  // pieces make of the same tokens; each lane takes the sum of both for four
  // tokens only: block 0's in the columns below 8, block 1's above. Maximum,
  // exponential and sum run on those, and the halves swap p's pieces for the
  // second matrix op: half the vector instructions of keeping both blocks in
  // both.
  auto compute = [&](StepData<BLK> &x, int s) {
    f32x4 acc[2];
#pragma unroll
    for (int j = 0; j < 2; j++) {
      acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (BLK) {
        const u32x2 c0 = codes_to_f16(x.k[j][0]), c1 = codes_to_f16(x.k[j][1]);
        const u32x2 c2 = codes_to_f16(x.k[j][2]), c3 = codes_to_f16(x.k[j][3]);
        acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
            __builtin_bit_cast(f16x8, u32x4{c0[0], c0[1], c1[0], c1[1]}),
            __builtin_bit_cast(f16x8, q0), acc[j], 0, 0, 0);
        acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
            __builtin_bit_cast(f16x8, u32x4{c2[0], c2[1], c3[0], c3[1]}),
            __builtin_bit_cast(f16x8, q1), acc[j], 0, 0, 0);
      } else {
        acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x.k[2 * j]),
                                                         __builtin_bit_cast(bf16x8, q0), acc[j], 0, 0, 0);
        acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x.k[2 * j + 1]),
                                                         __builtin_bit_cast(bf16x8, q1), acc[j], 0, 0, 0);
        if (FINE) {
          acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x.k[2 * j]),
                                                           __builtin_bit_cast(bf16x8, q2), acc[j], 0, 0, 0);
          acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x.k[2 * j + 1]),
                                                           __builtin_bit_cast(bf16x8, q3), acc[j], 0, 0, 0);
        }
      }
    }
    float t[4];
#pragma unroll
    for (int r = 0; r < 4; r++)
      t[r] = (low ? acc[1][r] : acc[0][r]) + swap8(low ? acc[0][r] : acc[1][r]);
    // The tokens of the block that are seen: all but in a sequence's last block
    // and in a window's first. The others get weight 0, and their values (never
    // written, or no longer seen) become 0.
    if (s == last_step || s == win_step || x.miss != 0) {
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const int i = 2 * s + j;
        const int blk = i < sp.first_blocks ? i : sp.win0 + i - sp.first_blocks;
        int hi = min(sp.L - blk * kBlockTokens, kBlockTokens);
        int lo = 0;
        if (a.window > 0 && i >= sp.first_blocks)
          lo = max(sp.L - a.window - blk * kBlockTokens, 0);
        if ((x.miss >> j) & 1)
          hi = 0;
        uint32_t keep = 0;
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const bool in = 4 * kg + r >= lo && 4 * kg + r < hi;
          keep |= in ? 0xffu << (8 * r) : 0u;
          if (!in && low == (j == 1))
            t[r] = -INFINITY;
        }
        if (BLK) {
#pragma unroll
          for (int nn = 0; nn < 4; nn++)
            x.v[j][nn] &= keep;
          if (hi == 0)
            x.sc[j] = f32x2{0.0f, 0.0f}; // (a missing block's scales are another block's)
        } else {
          const uint32_t m0 = (keep & 0xffu ? 0xffffu : 0u) | (keep & 0xff00u ? 0xffff0000u : 0u);
          const uint32_t m1 =
              (keep & 0xff0000u ? 0xffffu : 0u) | (keep & 0xff000000u ? 0xffff0000u : 0u);
#pragma unroll
          for (int h = 0; h < 2; h++) {
            u32x4 &v = x.v[2 * j + h];
            v = u32x4{v[0] & m0, v[1] & m1, v[2] & m0, v[3] & m1};
          }
        }
      }
    }
    // the scale of this lane's block (never 0: a masked score of -inf stays one; a NaN
    // stays a NaN)
    const float c =
        BLK ? __builtin_elementwise_maximum(qf * (low ? x.sc[1][0] : x.sc[0][0]), 1e-37f) : 1.0f;
    float mx = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])) * c;
    // The running maximum moves only when a score passes it by more than 8
    // (weights stay below 2^8); the test needs no cross-lane maximum, only the
    // move does (m is the same in the 8 lanes of a query head).
    if (__any(mx > st.m + 8.0f)) {
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      mx = fmaxf(mx, swap8(mx));
      const float m = fmaxf(st.m, mx);
      const float f = __builtin_amdgcn_exp2f(st.m - m);
      st.m = m;
      st.l *= f;
#pragma unroll
      for (int nn = 0; nn < 4; nn++)
        st.o[nn] *= f;
    }
    float p[4];
    const float vs = low ? x.sc[1][1] : x.sc[0][1];
#pragma unroll
    for (int r = 0; r < 4; r++) {
      p[r] = __builtin_amdgcn_exp2f(fmaf(t[r], c, -st.m));
      st.l += p[r];
      if (BLK)
        p[r] *= vs;
    }
    // p in bf16 and what that leaves, for the 4 tokens; the columns below 8 need
    // the first of both blocks, those above the second
    uint32_t hi[2], lo[2], w0[2], w1[2], t0[2], t1[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const float x0 = p[2 * k], x1 = p[2 * k + 1];
      hi[k] = f32x2_to_bf16_rne(x0, x1);
      const float r0 = x0 - __uint_as_float(hi[k] << 16), r1 = x1 - __uint_as_float(hi[k] & 0xffff0000u);
      lo[k] = f32x2_to_bf16_rne(r0, r1);
      const uint32_t got = __float_as_uint(swap8(__uint_as_float(low ? hi[k] : lo[k])));
      w0[k] = low ? got : hi[k];
      w1[k] = low ? lo[k] : got;
      if (FINE) { // the third of both blocks in the columns below 8
        const uint32_t th = f32x2_to_bf16_rne(r0 - __uint_as_float(lo[k] << 16),
                                              r1 - __uint_as_float(lo[k] & 0xffff0000u));
        const uint32_t from = __float_as_uint(swap8(__uint_as_float(th)));
        t0[k] = low ? 0 : th;
        t1[k] = low ? 0 : from;
      }
    }
    const bf16x8 pw = __builtin_bit_cast(bf16x8, u32x4{w0[0], w0[1], w1[0], w1[1]});
#pragma unroll
    for (int nn = 0; nn < 4; nn++) {
      u32x4 w;
      if (BLK) {
        const u32x2 y0 = fp8x4_to_bf16x4(x.v[0][nn]), y1 = fp8x4_to_bf16x4(x.v[1][nn]);
        w = u32x4{y0[0], y0[1], y1[0], y1[1]};
      } else {
        // half h = nn / 2 of each block, dims col + 32 h + 16 (nn % 2)
        const u32x4 y0 = x.v[nn / 2], y1 = x.v[2 + nn / 2];
        const int k = 2 * (nn & 1);
        w = u32x4{y0[k], y0[k + 1], y1[k], y1[k + 1]};
      }
      st.o[nn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), pw,
                                                         st.o[nn], 0, 0, 0);
      if (FINE)
        st.o[nn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            __builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, u32x4{t0[0], t0[1], t1[0], t1[1]}),
            st.o[nn], 0, 0, 0);
    }
  };

  for (int s = s0; s < s1; s += R) {
#pragma unroll
    for (int r = 0; r < R; r++) {
      if (s + r >= s1)
        break;
      const int2 next = ids_of(s + r + R);
      load(buf[(r + R - 1) % R], ids, s + r + R - 1);
      ids = next;
      compute(buf[r], s + r);
    }
  }
  if (bad && lane == 0 && a.dev_err)
    atomicOr(a.dev_err, GKV_DEVERR_BLOCK_ID);
  // the eight lanes of a query head hold its weights, its two columns the pieces
  // of its output
  st.l += __shfl_xor(st.l, 16);
  st.l += __shfl_xor(st.l, 32);
  st.l += swap8(st.l);
#pragma unroll
  for (int nn = 0; nn < 4; nn++)
#pragma unroll
    for (int r = 0; r < 4; r++)
      st.o[nn][r] += swap8(st.o[nn][r]);
  return st;
}

// The factor that turns sum p v (weights against the maximum m, sum l) into the
// output: 1 / (l + sink weight), 0 where nothing was seen.
__device__ __forceinline__ float out_factor(float m, float l, float sink2) {
  const float M = fmaxf(m, sink2);
  const float f = __builtin_amdgcn_exp2f(m - M);
  const float den = fmaf(l, f, __builtin_amdgcn_exp2f(sink2 - M));
  return den == 0.0f ? 0.0f : f / den; // (a NaN stays one)
}

__device__ __forceinline__ float sink_of(const KeptDecodeArgs &a, int g, int head) {
  return a.sinks ? a.sinks[g * a.G + head] * kLog2e : -INFINITY;
}

// The finished output of one (sequence, kv head), from the wave that holds it all.
__device__ __forceinline__ void put_whole(const KeptDecodeArgs &a, int b, int g, const State &st) {
  const int lane = threadIdx.x & 63, col = lane & 15, kg = lane >> 4;
  if (col >= a.G) // (at most 8: the high pieces' columns)
    return;
  const float f = out_factor(st.m, st.l, sink_of(a, g, col));
  const int64_t ob = (int64_t)b * a.out_stride + (int64_t)(g * a.G + col) * kHeadDim + 4 * kg;
#pragma unroll
  for (int nn = 0; nn < 4; nn++)
    put(a.out, ob + 16 * nn, st.o[nn] * f, a.out_bf16);
}

__device__ __forceinline__ void put_zeros(const KeptDecodeArgs &a, int64_t at, int n, int t, int nt) {
  for (int i = 4 * t; i < n; i += 4 * nt)
    put(a.out, at + i, f32x4{0.0f, 0.0f, 0.0f, 0.0f}, a.out_bf16);
}

} // namespace gkv
