// Decode attention for sequences that share their first blocks: samples and beams of one
// prompt, a batch behind one system prompt.
//
// The mathematics is that of kept_decode.hip (score = q.k / 8, softmax with the head's sink,
// out = sum p v); what differs is how often a byte is read. The first shared_blocks blocks of a
// group are read once for all its sequences: their query heads of a kv head are the columns
// of one matrix product, 16 a tile, so that those tokens cost 4 * 64 operations per column
// and token on the matrix cores instead of a stream from HBM per sequence. The blocks behind
// them are a sequence's own and stream as in kept_decode.hip.
//
// Two launches:
//   read     a workgroup of four waves takes tiles of a group's query heads and a part of its
//            shared blocks, or parts of some sequences' own blocks, and leaves (m, l, o) per
//            query head. Shared blocks are bound by the instructions that go with the matrix
//            ops, own blocks by HBM: both kinds of workgroups run side by side
//   join     the pieces of a sequence's query heads, in their order, the sink, the output
// A sequence shorter than the shared blocks is read on its own, so the prefix
// needs no mask.
//
// 8 kv heads of 8 query heads, bf16 outputs, both launches (in brackets: one kind of workgroup after
// the other, in launches of their own): 512 sequences of 129 .. 1025 own tokens behind a prompt of
// 2048, bf16, 147 us (170), 4.3 TB/s; 64 x 8 beams behind 256 .. 2048 tokens, codes, 58 (67); one
// request's four behind 2048 tokens 12 (13.6). 2 x 16 behind 27000, codes, fp32 outputs 61: 590 TF/s
// with the pieces of q and p; cutting those keeps the vector units longer than the matrix ones.
#include "kept_attend.hpp"
#include "lds_dma.hpp"

#include <algorithm>

namespace gkv {

constexpr int kSharedWaves = 4;

struct SharedArgs {
  KeptDecodeArgs a;
  const int32_t *cu_groups, *shared;
  int n_groups;
  int per, tiles_each;   // sequences of a prefix workgroup; tiles that a group has room for
  int splits, part_steps; // parts of a group's shared blocks, at most; steps of a part, at least
  int own_pieces, own_steps; // parts of a sequence's own blocks, at most; steps of one, at least
  float *ws_ml, *ws_o;   // [splits + own_pieces][B][Hq]: (m, l), o[64]
  int32_t *first;        // [B] shared blocks of a sequence that it does not read itself
  int prefix_wgs;        // of the first launch; behind them, those of own blocks
  int join_parts;        // waves per (sequence, kv head) of the second
};

// The last i in 0 .. n - 1 with key(i) <= x (key does not fall), -1 if there is none: by 256
// probes at a time, so that up to 256 groups take one round trip.
template <typename Key>
__device__ __forceinline__ int last_at_most(int n, int64_t x, Key key) {
  constexpr int P = 4;
  const int lane = threadIdx.x & 63;
  int64_t lo = 0, len = n;
  while (len > 0) {
    const int64_t step = (len + 64 * P - 1) / (64 * P);
    bool ok[P];
#pragma unroll
    for (int k = 0; k < P; k++) {
      const int64_t i = (lane + 64 * k) * step;
      ok[k] = i < len && key((int)(lo + i)) <= x;
    }
    int c = 0;
#pragma unroll
    for (int k = 0; k < P; k++)
      c += __popcll(__ballot(ok[k]));
    if (c == 0)
      return -1; // (only in the first round)
    lo += (c - 1) * step;
    if (step == 1)
      break;
    len = min(step, n - lo);
  }
  return uniform((int)lo);
}

// The group of sequence b (-1: none).
__device__ __forceinline__ int group_of(const SharedArgs &s, int b) {
  if (s.n_groups == 0)
    return -1;
  const int g = last_at_most(s.n_groups + 1, b, [&](int i) { return (int64_t)s.cu_groups[i]; });
  return g < 0 || g >= s.n_groups || s.cu_groups[g] > b || s.cu_groups[g + 1] <= b ? -1 : g;
}

// Whether group i's offsets are none: falling, or outside the batch. (What is read and written stays in
// range by itself; but parts of the prefix may then be nobody's, and what is joined instead anything.)
__device__ __forceinline__ bool offsets_fall(const SharedArgs &s, int64_t i) {
  if (i >= s.n_groups)
    return false;
  const int from = s.cu_groups[i], to = s.cu_groups[i + 1];
  return from < 0 || to < from || to > s.a.B;
}

__device__ __forceinline__ int shared_of(const SharedArgs &s, int grp) {
  return max(min(s.shared[grp], s.a.table_stride), 0);
}

// Steps of a part of n, and how many parts that makes.
__device__ __forceinline__ int part_steps(const SharedArgs &s, int n) {
  return max((n + s.splits - 1) / s.splits, s.part_steps);
}

// The same of a sequence's own blocks.
__device__ __forceinline__ int own_part_steps(const SharedArgs &s, int n) {
  return max((n + s.own_pieces - 1) / s.own_pieces, s.own_steps);
}

__device__ __forceinline__ int64_t piece_at(const SharedArgs &s, int i, int b) {
  return ((int64_t)i * s.a.B + b) * (s.a.n_kv_heads * s.a.G);
}

// ---- own ---------------------------------------------------------------------------------

// A workgroup's four waves take parts waves each of (sequence, kv head)s: the steps of a piece of its
// own blocks cut among them, joined in LDS. Alone, 512 sequences' 605 MB took 122 us (5 TB/s).
constexpr int kOwnBytes = kSharedWaves * (kPieceFloats + 2 * kHeads) * 4; // of LDS
template <bool BLK, bool FINE>
__device__ __forceinline__ void own_piece(const SharedArgs &s, int item, float *s_own) {
  const KeptDecodeArgs &a = s.a;
  float *s_o = s_own; // [4][kPieceFloats]
  float2 *s_ml = (float2 *)(s_own + kSharedWaves * kPieceFloats); // [4][kHeads]
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, kg = lane >> 4;
  const int pairs = a.B * a.n_kv_heads, each_wg = kSharedWaves / a.parts;
  const int wgs = (pairs + each_wg - 1) / each_wg; // of a piece
  const int slot = wave / a.parts, part = wave % a.parts;
  const int e = item / wgs, pair = item % wgs * each_wg + slot;
  const int b = min(pair, pairs - 1) / a.n_kv_heads, g = min(pair, pairs - 1) % a.n_kv_heads;
  const bool says = e == 0 && g == 0 && part == 0 && pair < pairs; // this wave speaks for its sequence
  // (and looks at some of the offsets, 64 of every 64 B: their loads go out before the others')
  bool none = false;
  if (says)
    none = offsets_fall(s, (int64_t)b * 64 + lane);
  const int len = uniform(a.seq_lens[b]), L = max(min(len, a.max_len), 0);
  const int grp = group_of(s, b), shared = grp < 0 ? 0 : uniform(shared_of(s, grp));
  const int first = L / kBlockTokens < shared ? 0 : shared;
  if (says) {
    for (int64_t i = (int64_t)(a.B + b) * 64 + lane; i < s.n_groups; i += (int64_t)a.B * 64)
      none |= offsets_fall(s, i);
    const bool wrong = __any(none) || len > a.max_len || (grp >= 0 && shared != s.shared[grp]);
    if (lane == 0) {
      s.first[b] = first;
      if (a.dev_err && wrong)
        atomicOr(a.dev_err, GKV_DEVERR_LENGTH);
    }
  }
  Span sp;
  sp.L = L;
  sp.first_blocks = sp.ring0 = 0;
  sp.win0 = first;
  sp.n_blocks = (L + kBlockTokens - 1) / kBlockTokens - first;
  const int n = span_steps(sp), each = own_part_steps(s, n);
  const int b0 = min(e * each, n), b1 = min(b0 + each, n);
  const bool ok = pair < pairs && b0 < b1;
  State st;
  st.m = kLowest;
  st.l = 0.0f;
#pragma unroll
  for (int nn = 0; nn < 4; nn++)
    st.o[nn] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const int s0 = b0 + part * (b1 - b0) / a.parts, s1 = b0 + (part + 1) * (b1 - b0) / a.parts;
  if (ok && s0 < s1)
    st = attend<BLK, 2, FINE>(a, b, g, sp, s0, s1);
  if (a.parts > 1) {
    if (ok && col < kHeads) {
#pragma unroll
      for (int nn = 0; nn < 4; nn++)
        *(f32x4 *)&s_o[wave * kPieceFloats + col * kHeadDim + 16 * nn + 4 * kg] = st.o[nn];
      if (kg == 0)
        s_ml[wave * kHeads + col] = float2{st.m, st.l};
    }
    __syncthreads();
  }
  if (!ok)
    return;
  const int64_t at = piece_at(s, s.splits + e, b) + g * a.G;
  if (a.parts == 1) {
    if (col < a.G) {
#pragma unroll
      for (int nn = 0; nn < 4; nn++)
        *(f32x4 *)(s.ws_o + (at + col) * kHeadDim + 16 * nn + 4 * kg) = st.o[nn];
      if (kg == 0)
        *(float2 *)(s.ws_ml + 2 * (at + col)) = float2{st.m, st.l};
    }
    return;
  }
  const int w0 = slot * a.parts;
  for (int i = part * 64 + lane; i < a.G * (kHeadDim / 4); i += a.parts * 64) {
    const int hh = i / (kHeadDim / 4);
    float m = kLowest, l = 0.0f;
    for (int p = 0; p < a.parts; p++)
      m = fmaxf(m, s_ml[(w0 + p) * kHeads + hh].x);
    f32x4 o{0.0f, 0.0f, 0.0f, 0.0f};
    for (int p = 0; p < a.parts; p++) {
      const float2 ml = s_ml[(w0 + p) * kHeads + hh];
      const float f = __builtin_amdgcn_exp2f(ml.x - m);
      l = fmaf(ml.y, f, l);
      o += *(const f32x4 *)&s_o[(w0 + p) * kPieceFloats + 4 * i] * f;
    }
    *(f32x4 *)(s.ws_o + at * kHeadDim + 4 * i) = o;
    if (i % (kHeadDim / 4) == 0)
      *(float2 *)(s.ws_ml + 2 * (at + hh)) = float2{m, l};
  }
}

// ---- prefix ----------------------------------------------------------------------------

// A workgroup's four waves hold 16 NT WQ query heads, WQ waves side by side; with WQ = 2 two pairs
// take a half of the tokens each and are joined at the end. The blocks come into
// LDS by loads of their own, in a ring of DP steps that the WQ waves share: a step is read from
// memory once for all of them, DP - 1 are under way while one is computed, and none of
// it takes registers. One barrier a step. A block's scales come the same way, and the block ids
// 64 at a time into a register's lanes: a scalar load in the loop would be waited for with
// the step's LDS reads, which share its counter (8 beams of 64 requests, codes: 65 us so).
// NT: tiles of 16 query heads per wave. Pieces of q and p as in kept_attend.hpp, whether a token is
// shared or not: q against codes two in fp16 (22 bits), against bf16 K two in bf16 (FINE three); p two in
// bf16 (FINE three), 2^-16 of a weight where the output's own rounding is 2^-8 of it. (One of
// each leaves a weight off by 2^-8, and a score against codes by 2^-11 of sum |q k| / 8, which grows with
// the score; 8 beams of 64 requests, codes, 55 us so, 58 with two.)
template <bool BLK, int NT, int WQ, bool FINE>
__global__ __launch_bounds__(64 * kSharedWaves)
__attribute__((amdgpu_waves_per_eu(NT == 1 ? (FINE ? 3 : 4) : BLK ? 3 : 2)))
void shared_read_kernel(SharedArgs s) {
  constexpr int D = kHeadDim, WT = kSharedWaves / WQ;
  constexpr int kHeadBytes = kBlockTokens * D * (BLK ? 1 : 2);
  constexpr int QP = BLK || !FINE ? 2 : 3, PP = FINE ? 3 : 2; // pieces of q, of p
  constexpr int kData = 4 * kHeadBytes;          // K and V of two blocks
  constexpr int kStage = kData + (BLK ? 256 : 0); // and their scales: K0, V0, K1, V1, in the first lanes
  constexpr int DP = WQ == 4 || BLK ? 3 : 2; // (deeper rings cost workgroups, and ran level)
  constexpr int UPW = kData / 1024 / WQ; // loads of a wave per step, 1 KB each
  constexpr int kRing = WT * DP * kStage, kJoin = (kSharedWaves / 2) * NT * 5 * 1024;
  __shared__ __attribute__((aligned(1024))) char s_mem[kRing > kJoin || WT == 1 ? kRing : kJoin];
  static_assert(sizeof(s_mem) >= kOwnBytes, "room for either kind");
  const KeptDecodeArgs &a = s.a;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), col = lane & 15, kg = lane >> 4;
  // (the prefix's workgroups, which are the longer ones, first, own blocks in the room beside them; both
  // in turn, 256 each, ran level)
  int item = blockIdx.x;
  if (item >= s.prefix_wgs) {
    own_piece<BLK, FINE>(s, item - s.prefix_wgs, (float *)s_mem);
    return;
  }
  const int g = item % a.n_kv_heads;
  item /= a.n_kv_heads;
  // Groups' tiles lie end to end, group i's from cu[i] / per + i on: room for all of them,
  // as every group wastes less than one. Workgroups take the groups' first tiles, part after part,
  // then the second ones and so on: the tiles that are not there come last. (In the order of the
  // tiles those that groups of one size leave empty, every second one, would leave every second CU
  // without work: 8 beams of 64 requests 64 us, 2 x 16 sequences 99.)
  const int order = item / s.n_groups, per = s.per, split = order % s.splits;
  const int tile = item % s.n_groups * s.tiles_each + order / s.splits;
  const int grp = last_at_most(s.n_groups, tile, [&](int i) {
    return (int64_t)(max(s.cu_groups[i], 0) / per) + i;
  });
  if (grp < 0)
    return;
  const int b0 = min(max(uniform(s.cu_groups[grp]), 0), a.B);
  const int b1 = min(max(uniform(s.cu_groups[grp + 1]), b0), a.B);
  const int first = uniform(shared_of(s, grp));
  if (first > a.max_len / kBlockTokens) // (no sequence is that long)
    return;
  const int n = (first + 1) / 2, each = part_steps(s, n);
  const int p0 = min(split * each, n), p1 = min(p0 + each, n);
  const int64_t at0 = b0 + (int64_t)(tile - (b0 / per + grp)) * per;
  if (p0 >= p1 || at0 < b0 || at0 >= b1)
    return;
  const int t0 = (int)at0, n_cols = min(b1 - t0, per) * a.G;
  const int part = wave / WQ, wq = wave % WQ;
  const int n_it = (p1 - p0 + WT - 1) / WT;
  const int s0 = min(p0 + part * n_it, p1), count = min(s0 + n_it, p1) - s0;

  // The block ids of this wave's steps, 32 steps in the lanes of a register, two registers in turn.
  const int32_t *trow = a.table + (int64_t)b0 * a.table_stride;
  auto ids_from = [&](int i) -> int { // ids of steps i .. i + 31
    const int at = 2 * (s0 + i) + lane;
    return at < 2 * (s0 + count) && at < first ? trow[at] : kNoBlock;
  };
  int ids_even = ids_from(0), ids_odd = kNoBlock;
  auto ids_of = [&](int i) -> int2 {
    const int v = i & 32 ? ids_odd : ids_even, at = 2 * (i & 31);
    return int2{__builtin_amdgcn_readlane(v, at), __builtin_amdgcn_readlane(v, at + 1)};
  };
  const char *k_head = a.kc + g * kHeadBytes, *v_head = a.vc + g * kHeadBytes;
  const uint32_t stride = (uint32_t)a.n_kv_heads * kHeadBytes;
  const uint32_t ring = lds_addr(s_mem) + part * DP * kStage;
  // 1: an id outside the pool (by its signs: scalar arithmetic, where a comparison becomes a mask)
  auto outside = [&](int id) -> uint32_t {
    return ((uint32_t)id | ((uint32_t)a.num_blocks - 1u - (uint32_t)id)) >> 31;
  };
  // A wave's loads of a step: units wq, wq + WQ, .. of its K0, K1, V0, V1 (KBs). A block that
  // is not there is read as block 0, whose values are dropped later.
  auto issue = [&](int i) {
    const int2 ids = ids_of(i);
#pragma unroll
    for (int x = 0; x < UPW; x++) {
      const int u = wq + x * WQ, v = u / (2 * kHeadBytes / 1024), j = u / (kHeadBytes / 1024) % 2;
      const int id = j ? ids.y : ids.x;
      const uint64_t off = (uint64_t)((uint32_t)id & (outside(id) - 1u)) * stride +
                           (BLK ? 0 : (uint32_t)(u % 2) * 1024u);
      // (codes of V: each lane's operand, in lane order)
      const uint32_t lane_off = BLK && v ? (uint32_t)(col * 4 + kg) * 16 : (uint32_t)lane * 16;
      dma16_at<false>((v ? v_head : k_head) + off, lane_off, ring + (i % DP) * kStage + u * 1024);
    }
    if (BLK && wq == 0) {
      const int id = lane & 2 ? ids.y : ids.x;
      dma4(a.scales + ((int64_t)((uint32_t)id & (outside(id) - 1u)) * a.n_kv_heads + g) * 2 + (lane & 1),
           s_mem + (part * DP + i % DP) * kStage + kData);
    }
  };
  // The columns' sequences and queries
  int seq[NT], head[NT], len[NT];
  bool on[NT], any = false;
  f32x4 qr[NT][4]; // dims 8 kg .. + 7 and 32 + 8 kg .. + 7
#pragma unroll
  for (int j = 0; j < NT; j++) {
    const int c = 16 * (wq * NT + j) + col;
    on[j] = c < n_cols;
    seq[j] = on[j] ? t0 + c / a.G : t0;
    head[j] = on[j] ? g * a.G + c % a.G : 0;
    len[j] = on[j] ? a.seq_lens[seq[j]] : 0;
    const f32x4 *qp = (const f32x4 *)(a.q + (int64_t)seq[j] * a.q_stride + head[j] * D + 8 * kg);
    qr[j][0] = qp[0];
    qr[j][1] = qp[1];
    qr[j][2] = qp[8];
    qr[j][3] = qp[9];
  }
#pragma unroll
  for (int i = 0; i < DP - 1; i++)
    if (i < count)
      issue(i);

#pragma unroll
  for (int j = 0; j < NT; j++) {
    len[j] = max(min(len[j], a.max_len), 0);
    on[j] &= len[j] >= first * kBlockTokens;
    any |= on[j];
  }
  const bool works = __any(any);
  u32x4 q[NT][QP][2];
  float qf[NT];
#pragma unroll
  for (int j = 0; j < NT; j++) {
    float x[2][8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      x[0][i] = on[j] ? qr[j][i / 4][i % 4] : 0.0f;
      x[1][i] = on[j] ? qr[j][2 + i / 4][i % 4] : 0.0f;
    }
    if (a.cos_tab && on[j]) {
      const f32x4 *cp = (const f32x4 *)(a.cos_tab + (int64_t)(len[j] - 1) * (D / 2) + 8 * kg);
      const f32x4 *np = (const f32x4 *)(a.sin_tab + (int64_t)(len[j] - 1) * (D / 2) + 8 * kg);
      const f32x4 an[4] = {cp[0], cp[1], np[0], np[1]};
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float y1 = x[0][i], y2 = x[1][i];
        x[0][i] = rope_first(y1, y2, an[i / 4][i % 4], an[2 + i / 4][i % 4]);
        x[1][i] = rope_second(y1, y2, an[i / 4][i % 4], an[2 + i / 4][i % 4]);
      }
    }
    qf[j] = 0.125f * kLog2e; // 1 / sqrt(64); exp -> exp2
    float down = qf[j];
    if (BLK) { // q * 2^-e has its largest element in [1, 2)
      float mx = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; i++)
        mx = fmaxf(mx, fmaxf(fabsf(x[0][i]), fabsf(x[1][i])));
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      const int e = min(max((int)(__float_as_uint(mx) >> 23), 27), 227);
      down = __uint_as_float((uint32_t)(254 - e) << 23);
      qf[j] *= __uint_as_float((uint32_t)e << 23);
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
      float rest[8];
#pragma unroll
      for (int i = 0; i < 8; i++)
        rest[i] = x[h][i] * down;
#pragma unroll
      for (int p = 0; p < QP; p++) {
        f16x8 yh;
        bf16x8 yb;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          if (BLK) {
            yh[i] = (_Float16)rest[i];
            rest[i] -= (float)yh[i];
          } else {
            yb[i] = (__bf16)rest[i];
            rest[i] -= (float)yb[i];
          }
        }
        q[j][p][h] = BLK ? __builtin_bit_cast(u32x4, yh) : __builtin_bit_cast(u32x4, yb);
      }
    }
  }

  State st[NT];
#pragma unroll
  for (int j = 0; j < NT; j++) {
    st[j].m = kLowest;
    st[j].l = 0.0f;
#pragma unroll
    for (int nn = 0; nn < 4; nn++)
      st[j].o[nn] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  // What the scores' sums begin with: 0, or -inf for a block that is not there.
  f32x4 begin[2] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
  uint32_t begun = 0; // bit j: so it is of block j
  auto compute = [&](int slot, uint32_t miss) {
      f32x2 sc[2] = {f32x2{0.0f, 0.0f}, f32x2{0.0f, 0.0f}};
      if (BLK) {
        const f32x2 *in_sc = (const f32x2 *)(s_mem + (part * DP + slot) * kStage + kData);
        sc[0] = in_sc[0];
        sc[1] = in_sc[1];
      }
      const u32x4 *in = (const u32x4 *)(s_mem + (part * DP + slot) * kStage) + lane;
      u32x4 x[BLK ? 2 : 4], y[BLK ? 2 : 4]; // K and V as they are stored
#pragma unroll
      for (int j = 0; j < (BLK ? 2 : 4); j++) {
        x[j] = in[j * 64];
        y[j] = in[(BLK ? 128 : 256) + j * 64];
      }
      if (miss != begun) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const float f = (miss >> j) & 1 ? -INFINITY : 0.0f;
          begin[j] = f32x4{f, f, f, f};
        }
        begun = miss;
      }
      if (miss != 0) { // (another block's values and scales)
#pragma unroll
        for (int j = 0; j < (BLK ? 2 : 4); j++)
          if ((miss >> (BLK ? j : j / 2)) & 1) {
            x[j] = y[j] = u32x4{0, 0, 0, 0};
            sc[j / (BLK ? 1 : 2)] = f32x2{0.0f, 0.0f};
          }
      }
      u32x4 k[2][2]; // [block][dims 0..31, 32..63]
#pragma unroll
      for (int j = 0; j < 2; j++)
        if (BLK) {
          const u32x2 c0 = codes_to_f16(x[j][0]), c1 = codes_to_f16(x[j][1]);
          const u32x2 c2 = codes_to_f16(x[j][2]), c3 = codes_to_f16(x[j][3]);
          k[j][0] = u32x4{c0[0], c0[1], c1[0], c1[1]};
          k[j][1] = u32x4{c2[0], c2[1], c3[0], c3[1]};
        } else {
          k[j][0] = x[2 * j];
          k[j][1] = x[2 * j + 1];
        }
      u32x4 v[4];
#pragma unroll
      for (int nn = 0; nn < 4; nn++) {
        if (BLK) {
          const u32x2 y0 = fp8x4_to_bf16x4(y[0][nn]), y1 = fp8x4_to_bf16x4(y[1][nn]);
          v[nn] = u32x4{y0[0], y0[1], y1[0], y1[1]};
        } else {
          const int k0 = 2 * (nn & 1);
          v[nn] = u32x4{y[nn / 2][k0], y[nn / 2][k0 + 1], y[2 + nn / 2][k0], y[2 + nn / 2][k0 + 1]};
        }
      }
      // All tiles' scores, then one test of their maxima, then weights and outputs tile by tile:
      // one tile's matrix ops under the next one's vector instructions.
      f32x4 acc[NT][2];
      float c[NT][2], mx[NT];
      bool moves = false;
#pragma unroll
      for (int j = 0; j < NT; j++) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
          acc[j][i] = begin[i];
#pragma unroll
          for (int p = 0; p < QP; p++)
#pragma unroll
            for (int h = 0; h < 2; h++)
              acc[j][i] = BLK ? __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                    __builtin_bit_cast(f16x8, k[i][h]),
                                    __builtin_bit_cast(f16x8, q[j][p][h]), acc[j][i], 0, 0, 0)
                              : __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                    __builtin_bit_cast(bf16x8, k[i][h]),
                                    __builtin_bit_cast(bf16x8, q[j][p][h]), acc[j][i], 0, 0, 0);
          // (never 0: a masked score of -inf stays one; a NaN stays a NaN)
          c[j][i] = BLK ? __builtin_elementwise_maximum(qf[j] * sc[i][0], 1e-37f) : 1.0f;
        }
        // (a NaN stays one, and the output becomes one)
        auto top = [](float x, float y) { return __builtin_elementwise_maximum(x, y); };
        const f32x4 &x0 = acc[j][0], &x1 = acc[j][1];
        mx[j] = top(top(top(x0[0], x0[1]), top(x0[2], x0[3])) * c[j][0],
                    top(top(x1[0], x1[1]), top(x1[2], x1[3])) * c[j][1]);
        moves |= mx[j] > st[j].m + 8.0f;
      }
      // (the running maximum moves only when a score passes it by more than 8)
      if (__any(moves)) {
#pragma unroll
        for (int j = 0; j < NT; j++) {
          State &t = st[j];
          float y = fmaxf(mx[j], __shfl_xor(mx[j], 16));
          y = fmaxf(y, __shfl_xor(y, 32));
          const float m = y > t.m + 8.0f ? y : t.m;
          const float f = __builtin_amdgcn_exp2f(t.m - m);
          t.m = m;
          t.l *= f;
#pragma unroll
          for (int nn = 0; nn < 4; nn++)
            t.o[nn] *= f;
        }
      }
#pragma unroll
      for (int j = 0; j < NT; j++) {
        State &t = st[j];
        float p[2][4];
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
          for (int r = 0; r < 4; r++) {
            p[i][r] = __builtin_amdgcn_exp2f(fmaf(acc[j][i][r], c[j][i], -t.m));
            t.l += p[i][r];
            if (BLK)
              p[i][r] *= sc[i][1];
          }
#pragma unroll
        for (int piece = 0; piece < PP; piece++) {
          u32x4 w;
#pragma unroll
          for (int i = 0; i < 2; i++)
#pragma unroll
            for (int r = 0; r < 2; r++) {
              const uint32_t y = f32x2_to_bf16_rne(p[i][2 * r], p[i][2 * r + 1]);
              w[2 * i + r] = y;
              if (piece + 1 < PP) {
                p[i][2 * r] -= __uint_as_float(y << 16);
                p[i][2 * r + 1] -= __uint_as_float(y & 0xffff0000u);
              }
            }
#pragma unroll
          for (int nn = 0; nn < 4; nn++)
            t.o[nn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                __builtin_bit_cast(bf16x8, v[nn]), __builtin_bit_cast(bf16x8, w), t.o[nn], 0, 0, 0);
        }
      }
    };
  uint32_t bad = 0;
  for (int i = 0; i < n_it; i++) {
    // this wave's loads of step i are done: the steps behind it may be under way
    if (i + DP - 1 > count)
      wait_vmcnt<0>();
    else if (BLK && wq == 0)
      wait_vmcnt<(DP - 2) * (UPW + 1)>();
    else
      wait_vmcnt<(DP - 2) * UPW>();
    lds_barrier(); // the others' too; and all are done with step i - 1, whose place is taken now
    if ((i & 31) == 0) { // the register that step i - 1 was the last to need
      const int next = i + 32 < count ? ids_from(i + 32) : kNoBlock;
      ids_even = i & 32 ? next : ids_even;
      ids_odd = i & 32 ? ids_odd : next;
    }
    if (i + DP - 1 < count)
      issue(i + DP - 1);
    if (i < count) {
      const int2 ids = ids_of(i);
      const uint32_t miss = outside(ids.x) | outside(ids.y) << 1;
      bad |= miss & (2 * (s0 + i) + 1 < first ? 3u : 1u);
      if (works)
        compute(i % DP, miss);
    }
  }
  if (bad != 0 && wq == 0 && lane == 0 && a.dev_err)
    atomicOr(a.dev_err, GKV_DEVERR_BLOCK_ID);
#pragma unroll
  for (int j = 0; j < NT; j++) {
    st[j].l += __shfl_xor(st[j].l, 16);
    st[j].l += __shfl_xor(st[j].l, 32);
  }

  if (WT == 2) { // the pair of the second half hands over to that of the first
    f32x4 *s_part = (f32x4 *)s_mem; // per wave [NT][5][64]: o, (m, l)
    lds_barrier(); // (the ring is free)
    if (part == 1) {
#pragma unroll
      for (int j = 0; j < NT; j++) {
#pragma unroll
        for (int nn = 0; nn < 4; nn++)
          s_part[((wq * NT + j) * 5 + nn) * 64 + lane] = st[j].o[nn];
        s_part[((wq * NT + j) * 5 + 4) * 64 + lane] = f32x4{st[j].m, st[j].l, 0.0f, 0.0f};
      }
    }
    lds_barrier();
    if (part == 0) {
#pragma unroll
      for (int j = 0; j < NT; j++) {
        const f32x4 *from = s_part + (wq * NT + j) * 5 * 64 + lane;
        const f32x4 ml = from[4 * 64];
        const float m = fmaxf(st[j].m, ml[0]);
        const float f0 = __builtin_amdgcn_exp2f(st[j].m - m), f1 = __builtin_amdgcn_exp2f(ml[0] - m);
        st[j].m = m;
        st[j].l = st[j].l * f0 + ml[1] * f1;
#pragma unroll
        for (int nn = 0; nn < 4; nn++)
          st[j].o[nn] = st[j].o[nn] * f0 + from[nn * 64] * f1;
      }
    }
  }
  if (part != 0)
    return;
#pragma unroll
  for (int j = 0; j < NT; j++)
    if (on[j]) {
      const int64_t at = piece_at(s, split, seq[j]) + head[j];
#pragma unroll
      for (int nn = 0; nn < 4; nn++)
        *(f32x4 *)(s.ws_o + at * D + 16 * nn + 4 * kg) = st[j].o[nn];
      if (kg == 0)
        *(float2 *)(s.ws_ml + 2 * at) = float2{st[j].m, st[j].l};
    }
}

// ---- join --------------------------------------------------------------------------------

// join_parts waves (1 or 4) per (sequence, kv head) go through its pieces, the prefix's and its own,
// 8 dims of a head a lane, and the first of them writes. Latency: 4 us for four sequences, 7.6 for
// 512 of three pieces (50 MB, which the launch before left in the caches).
__global__ __launch_bounds__(64 * kSharedWaves) void shared_join_kernel(SharedArgs s) {
  __shared__ f32x4 s_o[kSharedWaves][2][64];
  __shared__ float2 s_ml[kSharedWaves][64];
  const KeptDecodeArgs &a = s.a;
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int each_wg = kSharedWaves / s.join_parts, part = wave % s.join_parts;
  const int pairs = a.B * a.n_kv_heads, pair = blockIdx.x * each_wg + wave / s.join_parts;
  const int b = min(pair, pairs - 1) / a.n_kv_heads, g = min(pair, pairs - 1) % a.n_kv_heads;
  const int L = uniform(span_len(a, b)), first = uniform(s.first[b]);
  const int head = min(lane >> 3, a.G - 1), dim = 8 * (lane & 7);
  const int steps = (first + 1) / 2, own = ((L + kBlockTokens - 1) / kBlockTokens - first + 1) / 2;
  const int n_prefix = (steps + part_steps(s, steps) - 1) / part_steps(s, steps);
  const int n = n_prefix + (own + own_part_steps(s, own) - 1) / own_part_steps(s, own);
  float m = kLowest, l = 0.0f;
  f32x4 o[2] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
  auto join = [&](float2 with, f32x4 o0, f32x4 o1) {
    const float mn = fmaxf(m, with.x);
    const float f0 = __builtin_amdgcn_exp2f(m - mn), f1 = __builtin_amdgcn_exp2f(with.x - mn);
    m = mn;
    l = l * f0 + with.y * f1;
    o[0] = o[0] * f0 + o0 * f1;
    o[1] = o[1] * f0 + o1 * f1;
  };
  constexpr int A = 4; // pieces under way
  for (int i = part; i < n; i += A * s.join_parts) {
    float2 ml[A];
    f32x4 x[A][2];
#pragma unroll
    for (int k = 0; k < A; k++) {
      const int p = min(i + k * s.join_parts, n - 1);
      const int64_t at = piece_at(s, p < n_prefix ? p : s.splits + p - n_prefix, b) + g * a.G + head;
      ml[k] = *(const float2 *)(s.ws_ml + 2 * at);
      x[k][0] = *(const f32x4 *)(s.ws_o + at * kHeadDim + dim);
      x[k][1] = *(const f32x4 *)(s.ws_o + at * kHeadDim + dim + 4);
    }
#pragma unroll
    for (int k = 0; k < A; k++)
      if (i + k * s.join_parts < n)
        join(ml[k], x[k][0], x[k][1]);
  }
  if (s.join_parts > 1) {
    s_ml[wave][lane] = float2{m, l};
    s_o[wave][0][lane] = o[0];
    s_o[wave][1][lane] = o[1];
    __syncthreads();
    if (part == 0)
      for (int k = 1; k < s.join_parts; k++)
        join(s_ml[wave + k][lane], s_o[wave + k][0][lane], s_o[wave + k][1][lane]);
  }
  if (part != 0 || pair >= pairs || lane >= 8 * a.G)
    return;
  const float f = L > 0 ? out_factor(m, l, sink_of(a, g, head)) : 0.0f;
  const int64_t at = (int64_t)b * a.out_stride + (int64_t)(g * a.G + head) * kHeadDim + dim;
  put(a.out, at, o[0] * f, a.out_bf16);
  put(a.out, at + 4, o[1] * f, a.out_bf16);
}

// ---- host side ------------------------------------------------------------------------

// Pieces (times sequences) per kind, at most, or one per sequence: what the workspace holds, and no time
// lost (2 x 16 sequences behind 27000 tokens, codes: 512 67 us, 1024 56, 2048 56, 8192 55; 64 x 8 beams and
// 128 sequences on their own level).
constexpr int kSharedPieces = 2048;
// Steps of own blocks of a piece, at least (us with 18, 36, 72, 144, 288: 4 sequences of 8000 ..
// 16000 own tokens 27, 27, 24, 33, 53; 64 of 4000 .. 9000, codes, 117, 103, 101, 106, 101; 512 of 1000 .. 3000,
// codes, 235, 227, 219, 223, 223).
constexpr int kOwnSteps = 72;
// Steps of shared blocks of a part, at least, per wave that shares its tokens (us with 1, 2, 4, 8, 16: one
// request's four sequences behind 2048 tokens 12, 12, 12, 13, 18; 8 x 8 beams, codes, 25, 25, 22, 20, 28;
// 64 x 4 behind 64 .. 256 tokens 30, 30, 22, 23, 22).
constexpr int kLeastSteps = 4;

struct SharedPlan {
  int nt, wq, per, tiles_each;
  int64_t tiles;
  int splits, part_steps, own_pieces;
  size_t ml, o, total; // workspace (the sequences' first blocks come first)
};

static void shared_layout(SharedPlan &p, int32_t B, int64_t rows) {
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  p.ml = up((size_t)B * 4);
  p.o = p.ml + up((size_t)rows * 8);
  p.total = p.o + (size_t)rows * kHeadDim * 4;
}

static SharedPlan shared_plan(int32_t B, int32_t n_groups, int32_t n_q_heads, int32_t n_kv_heads,
                              int32_t max_shared, int32_t max_own, bool blk, bool fine) {
  SharedPlan p{};
  const int G = n_q_heads / n_kv_heads;
  const int64_t avg = n_groups > 0 ? std::max<int64_t>(1, ((int64_t)B + n_groups - 1) / n_groups) : 1;
  const int64_t cols = avg * G;
  // Shapes by the even group's query heads, us of both launches (64 groups of 256 .. 2048 shared
  // tokens and a token of each sequence's own, 8 kv heads, bf16 outputs): 32 heads, two waves of a tile 41 (codes
  // 38), four 48 (49); 64 heads, four waves of one tile 59 (57), two of two 54 (58), and with 1 .. 256
  // own tokens 84 (61) and 71 (58); 128 heads, four waves of two 85 (102), of one 88 (91);
  // 32 groups of 128 heads with own tokens 56 (60) and 66 (62).
  p.wq = cols <= 32 || (cols <= 64 && blk && !fine) ? 2 : 4;
  p.nt = cols <= 32 || (cols <= 64 && p.wq == 4) ? 1 : 2;
  p.per = 16 * p.nt * p.wq / G;
  // (as many tiles a group has room for as all of the even size need, and one)
  const int64_t each = (avg + p.per - 1) / p.per;
  p.tiles_each = (int)each + 1;
  p.tiles = p.tiles_each * (int64_t)n_groups;
  // Parts of equal steps, so that long groups have more of them and no workgroup is longer than
  // the rest; as many as the GPU holds at once, or fewer where a wave's registers are many: four waves
  // of two tiles 512 (512 sequences behind one prompt of 2048 tokens 145 us, 768 workgroups 168; codes
  // 110 and 120; 2 x 16 behind 27000, codes, 55 and 57), two of two 768 (8 beams of 64 requests, codes,
  // 58, 512 workgroups 59, 1024 63).
  const int64_t busy = std::max<int64_t>(n_groups * each * n_kv_heads, 1);
  const int64_t steps = ((int64_t)max_shared + 1) / 2;
  const int64_t wgs = p.nt == 2 ? (p.wq == 2 ? 768 : 512) : p.wq == 4 ? 2048 : 1024;
  const int64_t room = std::max<int64_t>(1, kSharedPieces / std::max(B, 1));
  const int least = kLeastSteps * (kSharedWaves / p.wq);
  const int64_t splits = std::min({wgs / busy, room, (steps + least - 1) / least});
  p.splits = (int)std::max<int64_t>(1, splits);
  p.part_steps = (int)std::max<int64_t>(least, (steps + p.splits - 1) / p.splits);
  const int64_t own_steps = (((int64_t)max_own + kBlockTokens - 1) / kBlockTokens + 1) / 2;
  p.own_pieces = (int)std::max<int64_t>(1, std::min((own_steps + kOwnSteps - 1) / kOwnSteps, room));
  shared_layout(p, B, (int64_t)(p.splits + p.own_pieces) * B * n_q_heads);
  return p;
}

// Room for any plan of up to B sequences, in groups of any number: of either kind at most room's
// pieces, which are kSharedPieces sequences' or one each, and at most what the steps make for each.
static size_t shared_room(int32_t B, int32_t n_q_heads, int32_t max_shared, int32_t max_own) {
  const int64_t most = std::max(kSharedPieces, B);
  const int64_t steps = ((int64_t)max_shared + 1) / 2;
  const int64_t own_steps = (((int64_t)max_own + kBlockTokens - 1) / kBlockTokens + 1) / 2;
  const int64_t splits = std::max<int64_t>(1, (steps + kLeastSteps - 1) / kLeastSteps);
  const int64_t own = std::max<int64_t>(1, (own_steps + kOwnSteps - 1) / kOwnSteps);
  SharedPlan p{};
  shared_layout(p, B, (std::min(most, splits * B) + std::min(most, own * B)) * n_q_heads);
  return p.total;
}

static bool shared_sizes_ok(int32_t B, int32_t n_groups, int32_t n_q_heads, int32_t n_kv_heads,
                            int32_t max_shared, int32_t max_own) {
  return B >= 0 && n_groups >= 0 && n_q_heads > 0 && n_kv_heads > 0 && n_kv_heads <= 8 &&
         n_q_heads % n_kv_heads == 0 && n_q_heads / n_kv_heads <= kHeads && max_shared >= 0 &&
         max_own >= 0;
}

template <bool BLK, bool FINE>
static void launch_read(const SharedPlan &p, dim3 grid, hipStream_t hs, const SharedArgs &s) {
  const dim3 block(64 * kSharedWaves);
  if (p.wq == 2 && p.nt == 1)
    hipLaunchKernelGGL((shared_read_kernel<BLK, 1, 2, FINE>), grid, block, 0, hs, s);
  else if (p.wq == 2) {
    if constexpr (BLK && !FINE)
      hipLaunchKernelGGL((shared_read_kernel<BLK, 2, 2, FINE>), grid, block, 0, hs, s);
  } else if (p.nt == 1)
    hipLaunchKernelGGL((shared_read_kernel<BLK, 1, 4, FINE>), grid, block, 0, hs, s);
  else
    hipLaunchKernelGGL((shared_read_kernel<BLK, 2, 4, FINE>), grid, block, 0, hs, s);
}

} // namespace gkv

extern "C" size_t gkv_shared_workspace_bytes(int32_t B, int32_t n_groups, int32_t n_q_heads,
                                             int32_t n_kv_heads, int32_t max_shared_blocks,
                                             int32_t max_own) {
  using namespace gkv;
  if (!shared_sizes_ok(B, n_groups, n_q_heads, n_kv_heads, max_shared_blocks, max_own))
    return 0;
  return shared_room(B, n_q_heads, max_shared_blocks, max_own);
}

extern "C" int gkv_shared_decode(void *stream, int32_t B, int32_t n_groups, const int32_t *cu_groups,
                                 const int32_t *shared_blocks, int32_t max_shared_blocks,
                                 int32_t max_own, int32_t n_q_heads, const float *q,
                                 int64_t q_stride, const float *cos_tab, const float *sin_tab,
                                 const int32_t *seq_lens, int32_t max_seq_len, gkv_cache_view cache,
                                 const float *sinks, void *workspace, size_t workspace_bytes,
                                 void *out, int64_t out_stride, int32_t out_dtype,
                                 uint32_t *dev_err) {
  using namespace gkv;
  if (B < 0 || n_groups < 0 || n_q_heads <= 0 || max_seq_len < 0 || max_shared_blocks < 0 ||
      max_own < 0 || !q || !seq_lens || !out || (n_groups > 0 && (!cu_groups || !shared_blocks)) ||
      (out_dtype != GKV_F32 && out_dtype != GKV_BF16) || (cos_tab == nullptr) != (sin_tab == nullptr))
    return GKV_ERR_ARG;
  int st = kept_check(cache, 0, 0, true);
  if (st != GKV_OK)
    return st;
  if (n_q_heads % cache.n_kv_heads != 0)
    return GKV_ERR_ARG;
  const int Hkv = cache.n_kv_heads, G = n_q_heads / Hkv;
  if (!shared_sizes_ok(B, n_groups, n_q_heads, Hkv, max_shared_blocks, max_own))
    return GKV_ERR_UNSUPPORTED;
  if (q_stride < (int64_t)n_q_heads * kHeadDim || out_stride < (int64_t)n_q_heads * kHeadDim)
    return GKV_ERR_ARG;
  // 16-byte loads of the query rows and the angles, 16- (bf16: 8-) byte stores
  if (q_stride % 4 != 0 || out_stride % 4 != 0 ||
      ((uintptr_t)q | (uintptr_t)cos_tab | (uintptr_t)sin_tab) % 16 != 0 ||
      (uintptr_t)out % (out_dtype == GKV_BF16 ? 8 : 16) != 0 ||
      ((uintptr_t)cu_groups | (uintptr_t)shared_blocks) % 4 != 0 || (uintptr_t)workspace % 16 != 0)
    return GKV_ERR_ARG;
  const bool blk = cache.v_format == GKV_KV_FP8_BLOCK, fine = out_dtype == GKV_F32;
  const SharedPlan p = shared_plan(B, n_groups, n_q_heads, Hkv, max_shared_blocks, max_own, blk, fine);
  SharedArgs s{};
  KeptDecodeArgs &a = s.a;
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
  a.max_len = (int)std::min<int64_t>(max_seq_len, kept_capacity(cache.table_stride, 0));
  a.sinks = sinks;
  a.B = B;
  a.G = G;
  a.n_kv_heads = Hkv;
  a.out = out;
  a.out_stride = out_stride;
  a.out_bf16 = out_dtype == GKV_BF16;
  a.dev_err = dev_err;
  s.cu_groups = cu_groups;
  s.shared = shared_blocks;
  s.n_groups = n_groups;
  s.per = p.per;
  s.tiles_each = p.tiles_each;
  s.splits = p.splits;
  s.part_steps = p.part_steps;
  s.own_pieces = p.own_pieces;
  s.own_steps = kOwnSteps;
  if (B == 0)
    return GKV_OK;
  // Waves per (sequence, head): more where few sequences are there (up to 512 waves in all, 1024, 2048, 4096:
  // 64 sequences of 100 .. 1000 own tokens, codes, 30 us, 22, 20, 20; 128 of them 35, 35, 28, 31), or long
  // ones (from 32 steps a wave on, 64, 128: 512 of 1000 .. 3000, codes, 225 us, 219, 231; 1024 of 100 .. 1200
  // 168, 173, 173). The join's waves the same way (four for up to 256 pairs, 1024: 64 sequences of
  // eight groups 23.7 us, 22.1; 512 level).
  const int64_t own = std::min<int64_t>((((int64_t)max_own + 15) / 16 + 1) / 2, kOwnSteps);
  const int64_t pairs = (int64_t)B * Hkv;
  a.parts = 1;
  while (a.parts < kSharedWaves && (2 * a.parts * pairs <= 2048 || own > 64 * a.parts))
    a.parts *= 2;
  s.join_parts = p.splits + p.own_pieces > 4 && pairs <= 1024 ? kSharedWaves : 1;
  const int64_t own_wgs = p.own_pieces * ((pairs * a.parts + kSharedWaves - 1) / kSharedWaves);
  const int64_t join_wgs = (pairs * s.join_parts + kSharedWaves - 1) / kSharedWaves;
  const int64_t prefix_wgs = p.tiles * p.splits * Hkv;
  if (pairs > INT32_MAX || !grid_fits(prefix_wgs + own_wgs, 64 * kSharedWaves))
    return GKV_ERR_UNSUPPORTED;
  if (!workspace || workspace_bytes < p.total)
    return GKV_ERR_WORKSPACE;
  s.first = (int32_t *)workspace;
  s.ws_ml = (float *)((char *)workspace + p.ml);
  s.ws_o = (float *)((char *)workspace + p.o);
  s.prefix_wgs = (int)prefix_wgs;
  hipStream_t hs = (hipStream_t)stream;
  const dim3 grid((unsigned)(prefix_wgs + own_wgs));
  if (blk && fine)
    launch_read<true, true>(p, grid, hs, s);
  else if (blk)
    launch_read<true, false>(p, grid, hs, s);
  else if (fine)
    launch_read<false, true>(p, grid, hs, s);
  else
    launch_read<false, false>(p, grid, hs, s);
  if ((st = launch_status("shared_read_kernel")))
    return st;
  hipLaunchKernelGGL(shared_join_kernel, dim3((unsigned)join_wgs), dim3(64 * kSharedWaves), 0, hs, s);
  return launch_status("shared_join_kernel");
}
