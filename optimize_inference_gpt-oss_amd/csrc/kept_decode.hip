// Decode attention over a cache of whole blocks: bf16, or e4m3 codes with one
// scale per block and kv head; every position, or a sliding window and the first
// tokens that stay visible.
//
// One query token per sequence and head: score = q.k / 8, softmax over the
// positions seen and (if given) the head's sink logit, out = sum p v. Each K and V
// byte is read once for the whole group of query heads; 2 * 64 * 2 operations a
// head and token against 128 (bf16: 256) bytes a kv head and token: bound by HBM.
//
// Matrix cores, 16x16 output, K = 32, the operand arrangement of the block
// layouts (kv_append.hpp): S^T = K Q^T and O^T += V^T P^T, columns 0..7 the high
// pieces of query head col's q and p, columns 8..15 the rest, added afterwards.
// Block codes enter without their scale, which is one number per block and
// wave: K's goes into the factor of the exponent, V's into the weights, so the
// stream costs no scale loads per token. Against codes q is split into fp16 pieces
// (e4m3 values are fp16 values; 22 bits of q, scaled by a power of two per head so
// that no range is lost), against bf16 K into bf16 pieces (16 bits); p always into
// bf16 pieces (its range is that of exp2). Two bf16 pieces leave up to 2^-18 of a
// value, 2^-9 of a bf16 output's own rounding; an fp32 output takes three, the
// third through matrix ops of its own (FINE).
//
// A step is two blocks (32 tokens). A wave takes the steps of one (sequence, kv
// head), loads the next step's blocks while it computes this one's, and leaves it
// to the other waves of its SIMD to cover the chain of matrix op, exponential,
// matrix op: 2 steps in registers, 4 waves per SIMD, with ranges 2 (3 or 4 steps
// and 3 or 5 waves measured the same or worse). Two ways to deal the steps out:
//   whole   contexts and windows that are not long: a (sequence, kv head) belongs
//           to 1 .. 8 waves of one workgroup, which cut its steps and merge in LDS.
//           One launch, no workspace. 512 sequences of 129 .. 2049 tokens (8 kv
//           heads, codes, 586 MB): 107 us, 5.5 TB/s; 97 windows of 4096 behind 64
//           (411 MB): 70 us, 5.9 TB/s.
//   ranges  the sequences laid end to end are cut into equal ranges, one per
//           wave; every workgroup finds its own range from the lengths
//           in its prologue. A sequence inside one range is finished there,
//           the pieces of the others go to the workspace and a second launch
//           merges them, a workgroup per range. 4 sequences of 129 .. 16384 tokens:
//           18 us, where one workgroup a sequence and head takes 43.
#include "kept.hpp"

#include <algorithm>

namespace gkv {

constexpr int kKeptAux = 2;            // nontemporal: each K/V byte is read once
constexpr int kHeads = 8;              // query heads per kv head, at most
// Range workgroups: one per CU, two waves a SIMD. Two per CU make twice the pieces
// and shorter ranges (us, 256 / 512 workgroups: 32 sequences of 129 .. 16384
// tokens 55.7 / 60.4, bf16 100 / 108; 4 of them 18.4 / 20.6, 22.1 / 28.3).
constexpr int kSplitWgs = 256;
constexpr int kMinRangeSteps = 4;      // steps per range, at least
constexpr int kPieceFloats = kHeads * kHeadDim;
constexpr int kPieceMl = 2 * kHeads;   // (m, l) of a piece's heads
constexpr float kLowest = -1e30f;      // the running maximum before any score (log2 units)
constexpr int kMergeThreads = 512;
constexpr int kMaxRanges = 8 * kSplitWgs; // one kv head: 8 ranges a workgroup

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

// ---- whole: one workgroup holds every step of its (sequence, kv head)s --------------

template <bool BLK, int R, int WPE, bool FINE>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(WPE)))
void kept_decode_whole_kernel(KeptDecodeArgs a) {
  __shared__ float s_o[8][kPieceFloats];
  __shared__ float2 s_ml[8][kHeads];
  const int n_groups = (a.n_kv_heads + a.heads_per_wg - 1) / a.heads_per_wg;
  const int b = blockIdx.x / n_groups;
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int slot = wave / a.parts, part = wave % a.parts;
  const int g = (int)(blockIdx.x % n_groups) * a.heads_per_wg + slot;
  const int len = uniform(a.seq_lens[b]);
  if (len > a.max_len && threadIdx.x == 0 && a.dev_err)
    atomicOr(a.dev_err, GKV_DEVERR_LENGTH);
  const Span sp = span_of(a, max(min(len, a.max_len), 0));
  const int n = span_steps(sp);
  const bool ok = g < a.n_kv_heads;
  if (n == 0) { // an empty sequence: zeros
    if (ok)
      put_zeros(a, (int64_t)b * a.out_stride + (int64_t)g * a.G * kHeadDim, a.G * kHeadDim,
                part * 64 + lane, a.parts * 64);
    return;
  }
  State st;
  if (ok) {
    const int s0 = part * n / a.parts, s1 = (part + 1) * n / a.parts;
    if (s0 < s1) {
      st = attend<BLK, R, FINE>(a, b, g, sp, s0, s1);
    } else {
      st.m = kLowest;
      st.l = 0.0f;
#pragma unroll
      for (int nn = 0; nn < 4; nn++)
        st.o[nn] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    if (a.parts == 1) {
      put_whole(a, b, g, st);
      return;
    }
    const int col = lane & 15, kg = lane >> 4;
    if (col < kHeads) {
#pragma unroll
      for (int nn = 0; nn < 4; nn++)
        *(f32x4 *)&s_o[wave][col * kHeadDim + 16 * nn + 4 * kg] = st.o[nn];
      if (kg == 0)
        s_ml[wave][col] = float2{st.m, st.l};
    }
  }
  if (a.parts == 1)
    return;
  __syncthreads();
  if (!ok)
    return;
  // the parts' sums against their common maximum, 4 dims a thread
  const int w0 = slot * a.parts;
  for (int e = part * 64 + lane; e < a.G * (kHeadDim / 4); e += a.parts * 64) {
    const int h = e / (kHeadDim / 4);
    float m = kLowest, l = 0.0f;
    for (int p = 0; p < a.parts; p++)
      m = fmaxf(m, s_ml[w0 + p][h].x);
    f32x4 o{0.0f, 0.0f, 0.0f, 0.0f};
    for (int p = 0; p < a.parts; p++) {
      const float f = __builtin_amdgcn_exp2f(s_ml[w0 + p][h].x - m);
      l = fmaf(s_ml[w0 + p][h].y, f, l);
      o += *(const f32x4 *)&s_o[w0 + p][4 * e] * f;
    }
    put(a.out, (int64_t)b * a.out_stride + (int64_t)g * a.G * kHeadDim + 4 * e,
        o * out_factor(m, l, sink_of(a, g, h)), a.out_bf16);
  }
}

// ---- ranges ----------------------------------------------------------------------
//
// (About 30 scalar registers of the prologue and the loop over sequences wait in lanes of a
// vector register while a wave is in its steps; nothing goes to memory.)

// Range r of the T steps cut into n (n <= 2048): floor(r T / n), in 32 bits.
__device__ __forceinline__ int range_begin(int r, int T, int n) {
  const uint32_t q = (uint32_t)T / (uint32_t)n, m = (uint32_t)T % (uint32_t)n;
  return (int)(r * q + r * m / (uint32_t)n);
}

// The range that holds step p.
__device__ __forceinline__ int range_of(int p, int T, int n) {
  return (int)(((int64_t)(p + 1) * n - 1) / T);
}

template <bool BLK, int R, int WPE, bool FINE>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(WPE)))
void kept_decode_split_kernel(KeptDecodeArgs a) {
  __shared__ int s_wave[8];
  __shared__ int s_b[8], s_c[8];
  const int t = threadIdx.x, lane = t & 63, wave = uniform(t >> 6), nt = blockDim.x;
  const int n_waves = nt >> 6, subs = n_waves / a.n_kv_heads; // ranges in this workgroup

  // Prefix sums of the sequences' steps: thread t holds sequences t * per ..
  const int per = (a.B + nt - 1) / nt;
  const int b0 = min(t * per, a.B), b1 = min(b0 + per, a.B);
  int mine = 0;
  bool over = false;
  for (int b = b0; b < b1; b++) {
    over |= a.seq_lens[b] > a.max_len;
    mine += span_steps(span_of(a, span_len(a, b)));
  }
  int incl = mine;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int v = __shfl_up(incl, off, 64);
    if (lane >= off)
      incl += v;
  }
  if (lane == 63)
    s_wave[wave] = incl;
  __syncthreads();
  int before = 0, T = 0;
  for (int w = 0; w < n_waves; w++) {
    const int v = s_wave[w];
    before += w < wave ? v : 0;
    T += v;
  }
  T = uniform(T);
  const int n = min(a.max_ranges, max(T / kMinRangeSteps, 1));
  const int r0 = blockIdx.x * subs;
  int c = before + incl - mine;
  // each of the workgroup's ranges: the sequence that holds its first step
  int at[8];
#pragma unroll
  for (int k = 0; k < 8; k++)
    at[k] = k < subs && r0 + k < n ? range_begin(r0 + k, T, n) : -1;
  for (int b = b0; b < b1; b++) {
    const int m = span_steps(span_of(a, span_len(a, b)));
#pragma unroll
    for (int k = 0; k < 8; k++)
      if (c <= at[k] && at[k] < c + m) {
        s_b[k] = b;
        s_c[k] = c;
        a.cuts[r0 + k] = int4{c < at[k] ? b : -1, c, c + m, T};
      }
    c += m;
  }
  if (t < subs && (r0 + t >= n || T == 0))
    a.cuts[r0 + t] = int4{-1, 0, 0, 0};
  if (blockIdx.x == 0 && over && a.dev_err)
    atomicOr(a.dev_err, GKV_DEVERR_LENGTH);
  // sequences without tokens: zeros
  for (int b = blockIdx.x; b < a.B; b += gridDim.x)
    if (a.seq_lens[b] <= 0 || a.max_len <= 0)
      put_zeros(a, (int64_t)b * a.out_stride, a.n_kv_heads * a.G * kHeadDim, t, nt);
  __syncthreads();

  const int sub = wave / a.n_kv_heads, g = wave % a.n_kv_heads;
  const int r = r0 + sub;
  if (r >= n || T == 0)
    return;
  const int rs = range_begin(r, T, n), re = range_begin(r + 1, T, n);
  int b = uniform(s_b[sub]), cb = uniform(s_c[sub]);
  while (cb < re) {
    const Span sp = span_of(a, uniform(span_len(a, b)));
    const int m = span_steps(sp);
    const int s0 = max(rs - cb, 0), s1 = min(re - cb, m);
    if (s0 < s1) {
      const State st = attend<BLK, R, FINE>(a, b, g, sp, s0, s1);
      if (s0 == 0 && s1 == m) {
        put_whole(a, b, g, st);
      } else {
        const int col = lane & 15, kg = lane >> 4;
        const int64_t piece = ((int64_t)r * 2 + (cb + s0 == rs ? 0 : 1)) * a.n_kv_heads + g;
        if (col < kHeads) {
          float *o = a.ws_o + piece * kPieceFloats + col * kHeadDim + 4 * kg;
#pragma unroll
          for (int nn = 0; nn < 4; nn++)
            *(f32x4 *)(o + 16 * nn) = st.o[nn];
          if (kg == 0)
            *(float2 *)(a.ws_ml + piece * kPieceMl + 2 * col) = float2{st.m, st.l};
        }
      }
    }
    cb += m;
    b++;
  }
}

// The pieces of a sequence that was cut: M = max m_i, out = sum o_i 2^(m_i - M) /
// (sum l_i 2^(m_i - M) + 2^(sink - M)). One workgroup per range, whose record
// (left by the split) names the sequence that the range starts inside of. A
// sequence of at most kMergeFew pieces is merged by the first such range's, a
// wave per kv head, every piece's loads at once. The kv heads of a longer one are
// dealt over all of them, a wave taking every eighth piece, four at a time, the waves
// joined in LDS. In one of more pieces than there are query heads each of those
// has a workgroup: 16 threads a piece (4 dims each), 32 pieces at a time, the first
// four of each thread loaded before the weights are known. Bound by latency: the
// record, then the pieces.
constexpr int kMergeFew = 4;
__global__ __launch_bounds__(kMergeThreads) void kept_decode_merge_kernel(KeptDecodeArgs a) {
  constexpr int D = kHeadDim, kWaves = kMergeThreads / 64, kGroups = kMergeThreads / 16;
  __shared__ float s_w[kMaxRanges];
  __shared__ float s_red[kWaves];
  __shared__ f32x4 s_o[kWaves][64][2];
  __shared__ float2 s_ml[kWaves][kHeads];
  const int4 cut = a.cuts[blockIdx.x];
  if (cut.x < 0)
    return;
  const int T = cut.w, n = min(a.max_ranges, max(T / kMinRangeSteps, 1)), b = cut.x;
  const int w0 = range_of(cut.y, T, n), np = range_of(cut.z - 1, T, n) - w0 + 1;
  const int inside = (int)blockIdx.x - w0 - 1;
  if (np <= kMergeFew && inside > 0)
    return;
  // the first piece is its range's last one, unless the sequence starts there
  const int first_slot = range_begin(w0, T, n) < cut.y ? 1 : 0;
  auto piece = [&](int i, int g) {
    return ((int64_t)(w0 + i) * 2 + (i == 0 ? first_slot : 0)) * a.n_kv_heads + g;
  };
  const int t = threadIdx.x, lane = t & 63, wave = uniform(t >> 6);
  if (np <= kMergeFew) {
    const int g = wave, h = lane >> 3, d0 = 8 * (lane & 7);
    if (g >= a.n_kv_heads || h >= a.G)
      return;
    float2 ml[kMergeFew];
    f32x4 x[kMergeFew][2];
#pragma unroll
    for (int i = 0; i < kMergeFew; i++) {
      const int64_t p = piece(min(i, np - 1), g);
      ml[i] = *(const float2 *)(a.ws_ml + p * kPieceMl + 2 * h);
      const f32x4 *o = (const f32x4 *)(a.ws_o + p * kPieceFloats + h * D + d0);
      x[i][0] = o[0];
      x[i][1] = o[1];
    }
    float m = kLowest, l = 0.0f;
#pragma unroll
    for (int i = 0; i < kMergeFew; i++)
      m = fmaxf(m, ml[i].x);
    f32x4 o0{0.0f, 0.0f, 0.0f, 0.0f}, o1{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kMergeFew; i++)
      if (i < np) {
        const float f = __builtin_amdgcn_exp2f(ml[i].x - m);
        l = fmaf(ml[i].y, f, l);
        o0 += x[i][0] * f;
        o1 += x[i][1] * f;
      }
    const float f = out_factor(m, l, sink_of(a, g, h));
    const int64_t ob = (int64_t)b * a.out_stride + (int64_t)(g * a.G + h) * D + d0;
    put(a.out, ob, o0 * f, a.out_bf16);
    put(a.out, ob + 4, o1 * f, a.out_bf16);
    return;
  }
  if (np - 1 < a.n_kv_heads * a.G) {
    const int h = lane >> 3, d0 = 8 * (lane & 7), hc = min(h, a.G - 1);
    for (int g = inside; g < a.n_kv_heads; g += np - 1) {
      float m = kLowest, l = 0.0f;
      f32x4 o0{0.0f, 0.0f, 0.0f, 0.0f}, o1{0.0f, 0.0f, 0.0f, 0.0f};
      for (int i0 = wave; i0 < np; i0 += 4 * kWaves) {
        float2 ml[4];
        f32x4 x[4][2];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int64_t p = piece(min(i0 + j * kWaves, np - 1), g);
          ml[j] = *(const float2 *)(a.ws_ml + p * kPieceMl + 2 * hc);
          const f32x4 *o = (const f32x4 *)(a.ws_o + p * kPieceFloats + hc * D + d0);
          x[j][0] = o[0];
          x[j][1] = o[1];
        }
        float mn = m;
#pragma unroll
        for (int j = 0; j < 4; j++)
          mn = fmaxf(mn, ml[j].x); // (a repeated last piece moves no maximum)
        const float f0 = __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= f0;
        o0 *= f0;
        o1 *= f0;
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (i0 + j * kWaves < np) {
            const float f = __builtin_amdgcn_exp2f(ml[j].x - m);
            l = fmaf(ml[j].y, f, l);
            o0 += x[j][0] * f;
            o1 += x[j][1] * f;
          }
      }
      __syncthreads(); // (the arrays may still be read for another head)
      s_o[wave][lane][0] = o0;
      s_o[wave][lane][1] = o1;
      if ((lane & 7) == 0)
        s_ml[wave][h] = float2{m, l};
      __syncthreads();
      // thread t < 128: 4 dims of query head t / 16
      const int th = t / 16;
      if (t < 128 && th < a.G) {
        float mt = kLowest, lt = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; w++)
          mt = fmaxf(mt, s_ml[w][th].x);
        f32x4 ot{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
          const float f = __builtin_amdgcn_exp2f(s_ml[w][th].x - mt);
          lt = fmaf(s_ml[w][th].y, f, lt);
          ot += s_o[w][t / 2][t & 1] * f;
        }
        put(a.out, (int64_t)b * a.out_stride + (int64_t)g * a.G * D + 4 * t,
            ot * out_factor(mt, lt, sink_of(a, g, th)), a.out_bf16);
      }
    }
    return;
  }
  const int grp = t >> 4, e = t & 15;
  for (int item = inside; item < a.n_kv_heads * a.G; item += np - 1) {
    const int g = item / a.G, h = item % a.G;
    auto load = [&](int i) {
      return *(const f32x4 *)(a.ws_o + piece(min(i, np - 1), g) * kPieceFloats + h * D + 4 * e);
    };
    f32x4 x[4];
#pragma unroll
    for (int j = 0; j < 4; j++)
      x[j] = load(grp + j * kGroups);
    // the common maximum, the pieces' weights, the sum
    float m = kLowest;
    for (int i = t; i < np; i += kMergeThreads)
      m = fmaxf(m, a.ws_ml[piece(i, g) * kPieceMl + 2 * h]);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1)
      m = fmaxf(m, __shfl_xor(m, off));
    __syncthreads(); // (the arrays may still be read for another head)
    if (lane == 0)
      s_red[wave] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; w++)
      m = fmaxf(m, s_red[w]);
    float l = 0.0f;
    for (int i = t; i < np; i += kMergeThreads) {
      const float2 ml = *(const float2 *)(a.ws_ml + piece(i, g) * kPieceMl + 2 * h);
      const float f = __builtin_amdgcn_exp2f(ml.x - m);
      s_w[i] = f;
      l = fmaf(ml.y, f, l);
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1)
      l += __shfl_xor(l, off);
    __syncthreads();
    if (lane == 0)
      s_red[wave] = l;
    f32x4 o{0.0f, 0.0f, 0.0f, 0.0f};
    for (int i = grp; i < np; i += 4 * kGroups) {
      f32x4 y[4];
#pragma unroll
      for (int j = 0; j < 4; j++)
        y[j] = i + 4 * kGroups < np ? load(i + (4 + j) * kGroups) : x[j];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if (i + j * kGroups < np)
          o += x[j] * s_w[i + j * kGroups];
        x[j] = y[j];
      }
    }
#pragma unroll
    for (int off = 16; off <= 32; off <<= 1)
#pragma unroll
      for (int r = 0; r < 4; r++)
        o[r] += __shfl_xor(o[r], off);
    if (lane < 16)
      s_o[wave][lane][0] = o;
    __syncthreads();
    if (t < 16) {
      o = s_o[0][t][0];
      l = s_red[0];
#pragma unroll
      for (int w = 1; w < kWaves; w++) {
        o += s_o[w][t][0];
        l += s_red[w];
      }
      put(a.out, (int64_t)b * a.out_stride + (int64_t)(g * a.G + h) * D + 4 * t,
          o * out_factor(m, l, sink_of(a, g, h)), a.out_bf16);
    }
  }
}

// ---- host side --------------------------------------------------------------------

// Steps of the longest sequence that a call with these bounds can meet.
static int64_t steps_bound(int32_t max_seq_len, int32_t kept, int32_t window) {
  int64_t blocks = ((int64_t)max_seq_len + kBlockTokens - 1) / kBlockTokens;
  if (window > 0)
    blocks = std::min<int64_t>(blocks, ((int64_t)kept + window) / kBlockTokens + 1);
  return (blocks + 1) / 2;
}

// Whole sequences or ranges. A wave takes about 1 us for a step (bf16: 1.2), eight
// share a sequence, so the longest one costs steps / 8 us whatever the rest do;
// ranges cost a second launch and their pieces, 5 to 10 us, but no sequence is
// longer than the others. Measured (us, whole / ranges, 8 heads, codes): 512
// sequences of 129 .. 2049 tokens 110 / 116 (bf16 192 / 209), 16 of them 10.7 /
// 17.0; 128 of 129 .. 4096 56 / 58, 8 of them 16.0 / 16.8 (bf16 19.1 / 18.0); 8 of
// 129 .. 8192 26 / 19, 4 of 129 .. 16384 43 / 18. A window of 4096 behind 16: 97
// sequences 68 / 76, 32 of them 25 / 34, 8 of them 18 / 16 (bf16 25 / 21).
constexpr int kWholeSteps = 72;      // whole whatever the number of sequences
constexpr int kWholeStepsMany = 144; // whole for this many (sequence, head)s
constexpr int kWholeMany = 96;
static bool use_whole(int32_t B, int32_t n_kv_heads, int32_t max_seq_len, int32_t kept,
                      int32_t window) {
  const int64_t steps = steps_bound(max_seq_len, kept, window);
  return steps <= kWholeSteps ||
         (steps <= kWholeStepsMany && (int64_t)B * n_kv_heads >= kWholeMany);
}

// Waves per (sequence, head) of the whole kernel. As many as take half the GPU's
// 4096 wave slots: more leave each wave too few steps (a window of 128: 512
// sequences 19 us with one, 32 with four) without reading faster. Contexts without a window differ
// in length, so there a wave gets at most 16 steps and the last sequences end
// sooner (512 sequences of 129 .. 2049 tokens: 126 us with one wave, 114, 108,
// 110 with 2, 4, 8; bf16 226, 206, 196, 189).
constexpr int kWholeWaves = 2048;
static int whole_parts(int32_t B, int32_t n_kv_heads, int64_t steps, int32_t window) {
  int parts = 1;
  while (parts < 8 && 2 * parts <= steps &&
         (2 * parts * (int64_t)B * n_kv_heads <= kWholeWaves ||
          (window == 0 && steps > 16 * parts)))
    parts *= 2;
  return parts;
}

static int range_subs(int n_kv_heads) { return 8 / n_kv_heads; }

struct KeptWorkspace {
  size_t ml, o, total; // (the ranges' records come first)
};
static KeptWorkspace kept_workspace(int32_t n_kv_heads) {
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  const size_t pieces = (size_t)kSplitWgs * range_subs(n_kv_heads) * 2 * n_kv_heads;
  KeptWorkspace w;
  w.ml = up((size_t)kSplitWgs * range_subs(n_kv_heads) * sizeof(int4));
  w.o = w.ml + up(pieces * kPieceMl * 4);
  w.total = w.o + pieces * kPieceFloats * 4;
  return w;
}

} // namespace gkv

extern "C" size_t gkv_kept_workspace_bytes(int32_t B, int32_t n_kv_heads, int32_t max_seq_len,
                                           int32_t kept, int32_t window) {
  using namespace gkv;
  // (what the call of any smaller batch needs too)
  if (B <= 0 || n_kv_heads <= 0 || n_kv_heads > 8 || max_seq_len < 0 || kept < 0 || window < 0 ||
      steps_bound(max_seq_len, kept, window) <= kWholeSteps)
    return 0;
  return kept_workspace(n_kv_heads).total;
}

extern "C" int gkv_kept_decode(void *stream, int32_t B, int32_t n_q_heads, const float *q,
                               int64_t q_stride, const float *cos_tab, const float *sin_tab,
                               const int32_t *seq_lens, int32_t max_seq_len, gkv_cache_view cache,
                               int32_t kept, int32_t window, const float *sinks, void *workspace,
                               size_t workspace_bytes, void *out, int64_t out_stride,
                               int32_t out_dtype, uint32_t *dev_err) {
  using namespace gkv;
  if (B < 0 || n_q_heads <= 0 || max_seq_len < 0 || !q || !seq_lens || !out ||
      (out_dtype != GKV_F32 && out_dtype != GKV_BF16) || (cos_tab == nullptr) != (sin_tab == nullptr))
    return GKV_ERR_ARG;
  int st = kept_check(cache, kept, window, true);
  if (st != GKV_OK)
    return st;
  if (n_q_heads % cache.n_kv_heads != 0)
    return GKV_ERR_ARG;
  const int G = n_q_heads / cache.n_kv_heads;
  if (cache.n_kv_heads > 8 || G > kHeads)
    return GKV_ERR_UNSUPPORTED;
  if (q_stride < (int64_t)n_q_heads * kHeadDim || out_stride < (int64_t)n_q_heads * kHeadDim)
    return GKV_ERR_ARG;
  // 16-byte loads of the query rows and the angles, 16- (bf16: 8-) byte stores
  if (q_stride % 4 != 0 || out_stride % 4 != 0 ||
      ((uintptr_t)q | (uintptr_t)cos_tab | (uintptr_t)sin_tab) % 16 != 0 ||
      (uintptr_t)out % (out_dtype == GKV_BF16 ? 8 : 16) != 0)
    return GKV_ERR_ARG;
  const int64_t steps = steps_bound(max_seq_len, kept, window);
  if ((int64_t)B * steps >= INT32_MAX || (int64_t)B * cache.n_kv_heads >= INT32_MAX)
    return GKV_ERR_UNSUPPORTED; // 32-bit step counts
  const bool blk = cache.v_format == GKV_KV_FP8_BLOCK;
  KeptDecodeArgs a{};
  a.q = q;
  a.q_stride = q_stride;
  a.cos_tab = cos_tab;
  a.sin_tab = sin_tab;
  a.seq_lens = seq_lens;
  a.kc = (const char *)cache.k;
  a.vc = (const char *)cache.v;
  a.scales = (const float *)cache.v_scale;
  a.table = cache.block_table;
  a.table_stride = cache.table_stride;
  a.num_blocks = cache.num_blocks;
  a.row = KeptRow{kept / kBlockTokens, cache.ring / kBlockTokens};
  a.window = window;
  a.max_len = (int)std::min<int64_t>(max_seq_len, kept_capacity(cache.table_stride, cache.ring) - 1);
  if (cache.ring == 0)
    a.max_len = (int)std::min<int64_t>(max_seq_len, kept_capacity(cache.table_stride, 0));
  a.sinks = sinks;
  a.B = B;
  a.G = G;
  a.n_kv_heads = cache.n_kv_heads;
  a.out = out;
  a.out_stride = out_stride;
  a.out_bf16 = out_dtype == GKV_BF16;
  a.dev_err = dev_err;
  hipStream_t s = (hipStream_t)stream;
  if (use_whole(B, a.n_kv_heads, max_seq_len, kept, window)) {
    if (B == 0)
      return GKV_OK;
    a.parts = whole_parts(B, a.n_kv_heads, steps, window);
    a.heads_per_wg = std::min(8 / a.parts, a.n_kv_heads);
    const int64_t wgs = (int64_t)B * ((a.n_kv_heads + a.heads_per_wg - 1) / a.heads_per_wg);
    const dim3 grid((unsigned)wgs), block(64 * a.parts * a.heads_per_wg);
    if (!grid_fits(wgs, block.x))
      return GKV_ERR_UNSUPPORTED;
    if (blk && a.out_bf16)
      hipLaunchKernelGGL((kept_decode_whole_kernel<true, 2, 4, false>), grid, block, 0, s, a);
    else if (blk)
      hipLaunchKernelGGL((kept_decode_whole_kernel<true, 2, 4, true>), grid, block, 0, s, a);
    else if (a.out_bf16)
      hipLaunchKernelGGL((kept_decode_whole_kernel<false, 2, 4, false>), grid, block, 0, s, a);
    else
      hipLaunchKernelGGL((kept_decode_whole_kernel<false, 2, 4, true>), grid, block, 0, s, a);
    return launch_status("kept_decode_whole_kernel");
  }
  const KeptWorkspace w = kept_workspace(a.n_kv_heads);
  if (B > 0 && (!workspace || workspace_bytes < w.total))
    return GKV_ERR_WORKSPACE;
  if ((uintptr_t)workspace % 16 != 0)
    return GKV_ERR_ARG;
  if (B == 0)
    return GKV_OK;
  const int subs = range_subs(a.n_kv_heads);
  a.max_ranges = kSplitWgs * subs;
  a.cuts = (int4 *)workspace;
  a.ws_ml = (float *)((char *)workspace + w.ml);
  a.ws_o = (float *)((char *)workspace + w.o);
  const dim3 block(64 * subs * a.n_kv_heads);
  if (blk && a.out_bf16)
    hipLaunchKernelGGL((kept_decode_split_kernel<true, 2, 2, false>), dim3(kSplitWgs), block, 0, s, a);
  else if (blk)
    hipLaunchKernelGGL((kept_decode_split_kernel<true, 2, 2, true>), dim3(kSplitWgs), block, 0, s, a);
  else if (a.out_bf16)
    hipLaunchKernelGGL((kept_decode_split_kernel<false, 2, 2, false>), dim3(kSplitWgs), block, 0, s, a);
  else
    hipLaunchKernelGGL((kept_decode_split_kernel<false, 2, 2, true>), dim3(kSplitWgs), block, 0, s, a);
  if ((st = launch_status("kept_decode_split_kernel")))
    return st;
  hipLaunchKernelGGL(kept_decode_merge_kernel, dim3((unsigned)a.max_ranges), dim3(kMergeThreads), 0, s,
                     a);
  return launch_status("kept_decode_merge_kernel");
}
