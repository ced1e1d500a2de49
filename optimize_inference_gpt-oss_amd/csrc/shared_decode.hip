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
//   prefix   a workgroup of four waves takes tiles of a group's query heads and a part of its
//            shared blocks, and leaves (m, l, o) per query head
//   own      a workgroup takes a sequence's own blocks (or, with long ones, its last part:
//            the others leave pieces in a launch before it), joins the pieces and writes
// A sequence shorter than the shared blocks is read on its own, so the prefix
// needs no mask.
#include "kept_attend.hpp"

#include <algorithm>

namespace gkv {

constexpr int kSharedWaves = 4;

struct SharedArgs {
  KeptDecodeArgs a;
  const int32_t *cu_groups, *shared;
  int n_groups;
  int seqs_per_wave, wq; // sequences of a wave's tiles; waves of a workgroup side by side on them
  int splits, min_steps; // parts of a group's shared blocks; steps of a part, at least
  int own_pieces, own_steps; // pieces before the last of a sequence's own blocks, at most; steps of one
  float *ws_ml, *ws_o;   // [splits + own_pieces][B][Hq]: (m, l), o[64]
};

// The last i in 0 .. n - 1 with key(i) <= x (key does not fall), -1 if there is none: by 64
// probes at a time.
template <typename Key>
__device__ __forceinline__ int last_at_most(int n, int64_t x, Key key) {
  const int lane = threadIdx.x & 63;
  int64_t lo = 0, len = n;
  while (len > 0) {
    const int64_t step = (len + 63) / 64, i = lo + lane * step;
    const bool ok = lane * step < len && key((int)i) <= x;
    const int c = __popcll(__ballot(ok));
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

__device__ __forceinline__ int shared_of(const SharedArgs &s, int grp) {
  return max(min(s.shared[grp], s.a.table_stride), 0);
}

// Steps of a part of n, and how many parts that makes.
__device__ __forceinline__ int part_steps(const SharedArgs &s, int n) {
  return max((n + s.splits - 1) / s.splits, s.min_steps);
}

__device__ __forceinline__ int64_t piece_at(const SharedArgs &s, int i, int b) {
  return ((int64_t)i * s.a.B + b) * (s.a.n_kv_heads * s.a.G);
}

// ---- prefix ----------------------------------------------------------------------------

// NT: tiles of 16 query heads per wave. Pieces of q: bf16 K two in bf16 (FINE three), codes one
// in fp16 (FINE two); p: one in bf16 (FINE three). A bf16 output's own rounding is off by at most
// 2^-8 of it; so is a weight here, each at random, and q's 11 (16) bits leave far less.
template <bool BLK, int NT, bool FINE>
__global__ __launch_bounds__(64 * kSharedWaves) __attribute__((amdgpu_waves_per_eu(FINE ? 1 : 2)))
void shared_prefix_kernel(SharedArgs s) {
  constexpr int D = kHeadDim;
  constexpr int kHeadBytes = kBlockTokens * D * (BLK ? 1 : 2);
  constexpr int QP = BLK ? (FINE ? 2 : 1) : (FINE ? 3 : 2);
  const KeptDecodeArgs &a = s.a;
  extern __shared__ f32x4 s_part[]; // per wave of a tile's upper half [NT][5][64]: o, (m, l)
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), col = lane & 15, kg = lane >> 4;
  int item = blockIdx.x;
  const int g = item % a.n_kv_heads;
  item /= a.n_kv_heads;
  const int split = item % s.splits, tile = item / s.splits;
  const int per = s.seqs_per_wave * s.wq;
  // Groups' tiles lie end to end, group i's from cu[i] / per + i on: room for all of them,
  // as every group wastes less than one.
  const int grp = last_at_most(s.n_groups, tile, [&](int i) {
    return (int64_t)(max(s.cu_groups[i], 0) / per) + i;
  });
  if (grp < 0)
    return;
  const int b0 = min(max(uniform(s.cu_groups[grp]), 0), a.B);
  const int b1 = min(max(uniform(s.cu_groups[grp + 1]), b0), a.B);
  const int first = uniform(shared_of(s, grp));
  const int n = (first + 1) / 2, each = part_steps(s, n);
  const int p0 = min(split * each, n), p1 = min(p0 + each, n);
  const int64_t at0 = b0 + (int64_t)(tile - (b0 / per + grp)) * per;
  if (p0 >= p1 || at0 < b0 || at0 >= b1)
    return;
  const int t0 = (int)at0;
  const int wt = kSharedWaves / s.wq, part = wave / s.wq;
  const int seq0 = t0 + (wave % s.wq) * s.seqs_per_wave;
  const int n_cols = min(max(b1 - seq0, 0), s.seqs_per_wave) * a.G;
  const int s0 = p0 + part * (p1 - p0) / wt, s1 = p0 + (part + 1) * (p1 - p0) / wt;

  // The columns' sequences and queries
  int seq[NT], head[NT], len[NT];
  bool on[NT], any = false;
#pragma unroll
  for (int j = 0; j < NT; j++) {
    const int c = 16 * j + col;
    on[j] = c < n_cols;
    seq[j] = on[j] ? seq0 + c / a.G : seq0;
    head[j] = on[j] ? g * a.G + c % a.G : 0;
    len[j] = 0;
    if (on[j]) {
      len[j] = span_len(a, seq[j]);
      on[j] = len[j] >= first * kBlockTokens;
    }
    any |= on[j];
  }
  const bool works = __any(any) && s0 < s1;
  u32x4 q[NT][QP][2];
  float qf[NT];
#pragma unroll
  for (int j = 0; j < NT; j++) {
    float x[2][8];
#pragma unroll
    for (int i = 0; i < 8; i++)
      x[0][i] = x[1][i] = 0.0f;
    if (on[j]) {
      const f32x4 *qp = (const f32x4 *)(a.q + (int64_t)seq[j] * a.q_stride + head[j] * D + 8 * kg);
      const f32x4 qr[4] = {qp[0], qp[1], qp[8], qp[9]};
#pragma unroll
      for (int i = 0; i < 8; i++) {
        x[0][i] = qr[i / 4][i % 4];
        x[1][i] = qr[2 + i / 4][i % 4];
      }
      if (a.cos_tab) {
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

  if (works) {
    const uint32_t k_off = lane * 16, v_off = BLK ? (col * 4 + kg) * 16 : lane * 16;
    const ScalarI32 trow = (ScalarI32)a.table + (int64_t)b0 * a.table_stride;
    bool bad = false;
    auto ids_of = [&](int i) -> int2 {
      int2 r{kNoBlock, kNoBlock};
      if (i < s1) {
        r.x = trow[2 * i];
        if (2 * i + 1 < first)
          r.y = trow[2 * i + 1];
      }
      return r;
    };
    const char *k_head = a.kc + g * kHeadBytes, *v_head = a.vc + g * kHeadBytes;
    const char *s_head = (const char *)a.scales + g * 8;
    const uint32_t stride = (uint32_t)a.n_kv_heads * kHeadBytes;
    auto load = [&](StepData<BLK> &x, int2 ids, int i) {
      x.miss = 0;
      const bool one = i < s1, two = one && 2 * i + 1 < first;
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const int id = uniform(j ? ids.y : ids.x);
        const bool ok = (uint32_t)id < (uint32_t)a.num_blocks;
        bad |= !ok && (j ? two : one);
        x.miss |= ok ? 0u : 1u << j;
        const uint64_t off = (uint64_t)(ok ? (uint32_t)id : 0u) * stride;
        const __amdgpu_buffer_rsrc_t kr = head_rsrc(k_head + off, ok ? kHeadBytes : 0);
        const __amdgpu_buffer_rsrc_t vr = head_rsrc(v_head + off, ok ? kHeadBytes : 0);
        if (BLK) {
          x.sc[j] = *(ScalarF2)(s_head + off / 128);
          x.k[j] = __builtin_amdgcn_raw_buffer_load_b128(kr, k_off, 0, 0);
          x.v[j] = __builtin_amdgcn_raw_buffer_load_b128(vr, v_off, 0, 0);
        } else {
#pragma unroll
          for (int h = 0; h < 2; h++) {
            x.k[2 * j + h] = __builtin_amdgcn_raw_buffer_load_b128(kr, k_off + h * 1024, 0, 0);
            x.v[2 * j + h] = __builtin_amdgcn_raw_buffer_load_b128(vr, v_off + h * 1024, 0, 0);
          }
        }
      }
    };
    auto compute = [&](StepData<BLK> &x) {
      u32x4 k[2][2]; // [block][dims 0..31, 32..63]
#pragma unroll
      for (int j = 0; j < 2; j++)
        if (BLK) {
          const u32x2 c0 = codes_to_f16(x.k[j][0]), c1 = codes_to_f16(x.k[j][1]);
          const u32x2 c2 = codes_to_f16(x.k[j][2]), c3 = codes_to_f16(x.k[j][3]);
          k[j][0] = u32x4{c0[0], c0[1], c1[0], c1[1]};
          k[j][1] = u32x4{c2[0], c2[1], c3[0], c3[1]};
        } else {
          k[j][0] = x.k[2 * j];
          k[j][1] = x.k[2 * j + 1];
        }
      if (x.miss != 0) { // a block that is not there: its values become 0, its weights too
#pragma unroll
        for (int j = 0; j < 2; j++)
          if ((x.miss >> j) & 1) {
            x.sc[j] = f32x2{0.0f, 0.0f};
            if (BLK)
              x.v[j] = u32x4{0, 0, 0, 0};
            else
              x.v[2 * j] = x.v[2 * j + 1] = u32x4{0, 0, 0, 0};
          }
      }
      u32x4 v[4];
#pragma unroll
      for (int nn = 0; nn < 4; nn++) {
        if (BLK) {
          const u32x2 y0 = fp8x4_to_bf16x4(x.v[0][nn]), y1 = fp8x4_to_bf16x4(x.v[1][nn]);
          v[nn] = u32x4{y0[0], y0[1], y1[0], y1[1]};
        } else {
          const u32x4 y0 = x.v[nn / 2], y1 = x.v[2 + nn / 2];
          const int k0 = 2 * (nn & 1);
          v[nn] = u32x4{y0[k0], y0[k0 + 1], y1[k0], y1[k0 + 1]};
        }
      }
#pragma unroll
      for (int j = 0; j < NT; j++) {
        f32x4 acc[2];
        float c[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
          acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int p = 0; p < QP; p++)
#pragma unroll
            for (int h = 0; h < 2; h++)
              acc[i] = BLK ? __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                 __builtin_bit_cast(f16x8, k[i][h]),
                                 __builtin_bit_cast(f16x8, q[j][p][h]), acc[i], 0, 0, 0)
                           : __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                 __builtin_bit_cast(bf16x8, k[i][h]),
                                 __builtin_bit_cast(bf16x8, q[j][p][h]), acc[i], 0, 0, 0);
          if ((x.miss >> i) & 1)
            acc[i] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          // (never 0: a masked score of -inf stays one; a NaN stays a NaN)
          c[i] = BLK ? __builtin_elementwise_maximum(qf[j] * x.sc[i][0], 1e-37f) : 1.0f;
        }
        State &t = st[j];
        float mx = fmaxf(fmaxf(fmaxf(acc[0][0], acc[0][1]), fmaxf(acc[0][2], acc[0][3])) * c[0],
                         fmaxf(fmaxf(acc[1][0], acc[1][1]), fmaxf(acc[1][2], acc[1][3])) * c[1]);
        // (the running maximum moves only when a score passes it by more than 8)
        if (__any(mx > t.m + 8.0f)) {
          mx = fmaxf(mx, __shfl_xor(mx, 16));
          mx = fmaxf(mx, __shfl_xor(mx, 32));
          const float m = fmaxf(t.m, mx);
          const float f = __builtin_amdgcn_exp2f(t.m - m);
          t.m = m;
          t.l *= f;
#pragma unroll
          for (int nn = 0; nn < 4; nn++)
            t.o[nn] *= f;
        }
        float p[2][4];
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
          for (int r = 0; r < 4; r++) {
            p[i][r] = __builtin_amdgcn_exp2f(fmaf(acc[i][r], c[i], -t.m));
            t.l += p[i][r];
            if (BLK)
              p[i][r] *= x.sc[i][1];
          }
#pragma unroll
        for (int piece = 0; piece < (FINE ? 3 : 1); piece++) {
          u32x4 w;
#pragma unroll
          for (int i = 0; i < 2; i++)
#pragma unroll
            for (int r = 0; r < 2; r++) {
              const uint32_t y = f32x2_to_bf16_rne(p[i][2 * r], p[i][2 * r + 1]);
              w[2 * i + r] = y;
              if (FINE) {
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
    StepData<BLK> buf[2];
    int2 ids = ids_of(s0);
    load(buf[0], ids, s0);
    ids = ids_of(s0 + 1);
    for (int i = s0; i < s1; i += 2) {
#pragma unroll
      for (int r = 0; r < 2; r++) {
        if (i + r >= s1)
          break;
        const int2 next = ids_of(i + r + 2);
        load(buf[r ^ 1], ids, i + r + 1);
        ids = next;
        compute(buf[r]);
      }
    }
    if (bad && lane == 0 && a.dev_err)
      atomicOr(a.dev_err, GKV_DEVERR_BLOCK_ID);
#pragma unroll
    for (int j = 0; j < NT; j++) {
      st[j].l += __shfl_xor(st[j].l, 16);
      st[j].l += __shfl_xor(st[j].l, 32);
    }
  }

  // the waves of a tile that split its tokens: the upper half of them hands over to the lower,
  // until one is left
  for (int half = wt / 2; half >= 1; half /= 2) {
    const int place = (part - half) * s.wq + wave % s.wq;
    if (part >= half && part < 2 * half) {
#pragma unroll
      for (int j = 0; j < NT; j++) {
#pragma unroll
        for (int nn = 0; nn < 4; nn++)
          s_part[((place * NT + j) * 5 + nn) * 64 + lane] = st[j].o[nn];
        s_part[((place * NT + j) * 5 + 4) * 64 + lane] = f32x4{st[j].m, st[j].l, 0.0f, 0.0f};
      }
    }
    __syncthreads();
    if (part < half) {
#pragma unroll
      for (int j = 0; j < NT; j++) {
        const f32x4 *from = s_part + (wave * NT + j) * 5 * 64 + lane; // (place of wave + half wq)
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
    __syncthreads();
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

// ---- own ---------------------------------------------------------------------------------

// parts waves of a workgroup per (sequence, kv head): the steps of its own blocks cut among
// them, the pieces of the prefix (and of earlier own blocks) too; joined in LDS. LAST: the
// last part, which joins and writes; else part blockIdx.y, which leaves a piece.
template <bool BLK, bool FINE, bool LAST>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(4)))
void shared_own_kernel(SharedArgs s) {
  __shared__ float s_o[8][kPieceFloats];
  __shared__ float2 s_ml[8][kHeads];
  const KeptDecodeArgs &a = s.a;
  const int n_wg = (a.n_kv_heads + a.heads_per_wg - 1) / a.heads_per_wg;
  const int b = blockIdx.x / n_wg;
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, kg = lane >> 4;
  const int slot = wave / a.parts, part = wave % a.parts;
  const int g = (int)(blockIdx.x % n_wg) * a.heads_per_wg + slot;
  const bool ok = g < a.n_kv_heads;
  const int len = uniform(a.seq_lens[b]), L = max(min(len, a.max_len), 0);
  if (LAST && len > a.max_len && threadIdx.x == 0 && a.dev_err)
    atomicOr(a.dev_err, GKV_DEVERR_LENGTH);
  const int Hq = a.n_kv_heads * a.G;
  if (L == 0) {
    if (LAST && ok)
      put_zeros(a, (int64_t)b * a.out_stride + (int64_t)g * a.G * kHeadDim, a.G * kHeadDim,
                part * 64 + lane, a.parts * 64);
    return;
  }
  const int grp = group_of(s, b);
  int first = grp < 0 ? 0 : uniform(shared_of(s, grp));
  if (LAST && grp >= 0 && threadIdx.x == 0 && first != s.shared[grp] && a.dev_err)
    atomicOr(a.dev_err, GKV_DEVERR_LENGTH);
  if (L < first * kBlockTokens)
    first = 0;
  Span sp;
  sp.L = L;
  sp.first_blocks = sp.ring0 = 0;
  sp.win0 = first;
  sp.n_blocks = (L + kBlockTokens - 1) / kBlockTokens - first;
  // this workgroup's steps: part e of own_pieces + 1
  const int n = span_steps(sp);
  const int each = max((n + s.own_pieces) / (s.own_pieces + 1), s.own_steps);
  const int before = n > 0 ? (n - 1) / each : 0; // pieces before the last
  const int e = LAST ? before : (int)blockIdx.y;
  if (!LAST && e >= before)
    return;
  const int b0 = e * each, b1 = min(b0 + each, n);
  State st;
  st.m = kLowest;
  st.l = 0.0f;
#pragma unroll
  for (int nn = 0; nn < 4; nn++)
    st.o[nn] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (ok) {
    if (LAST) { // the pieces first, into LDS: head lane / 8, dims 8 (lane % 8) ..
      float pm = kLowest, pl = 0.0f;
      f32x4 po[2] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
      const int h = lane >> 3, d0 = 8 * (lane & 7);
      const int steps = (first + 1) / 2;
      const int n_prefix = first > 0 ? (steps + part_steps(s, steps) - 1) / part_steps(s, steps) : 0;
      const int hc = g * a.G + min(h, a.G - 1);
      for (int i = part; i < n_prefix + before; i += a.parts) {
        const int64_t at = piece_at(s, i < n_prefix ? i : s.splits + i - n_prefix, b) + hc;
        const float2 ml = *(const float2 *)(s.ws_ml + 2 * at);
        const f32x4 *o = (const f32x4 *)(s.ws_o + at * kHeadDim + d0);
        const f32x4 x0 = o[0], x1 = o[1];
        const float m = fmaxf(pm, ml.x);
        const float f0 = __builtin_amdgcn_exp2f(pm - m), f1 = __builtin_amdgcn_exp2f(ml.x - m);
        pm = m;
        pl = pl * f0 + ml.y * f1;
        po[0] = po[0] * f0 + x0 * f1;
        po[1] = po[1] * f0 + x1 * f1;
      }
      f32x4 *o = (f32x4 *)&s_o[wave][h * kHeadDim + d0];
      o[0] = po[0];
      o[1] = po[1];
      if ((lane & 7) == 0)
        s_ml[wave][h] = float2{pm, pl};
    }
    const int s0 = b0 + part * (b1 - b0) / a.parts, s1 = b0 + (part + 1) * (b1 - b0) / a.parts;
    if (s0 < s1)
      st = attend<BLK, 2, FINE>(a, b, g, sp, s0, s1);
    __builtin_amdgcn_wave_barrier(); // (a wave's LDS accesses keep their order)
    if (col < kHeads) {
      if (LAST) { // the pieces onto what the blocks gave
        const float2 ml = s_ml[wave][col];
        const float m = fmaxf(st.m, ml.x);
        const float f0 = __builtin_amdgcn_exp2f(st.m - m), f1 = __builtin_amdgcn_exp2f(ml.x - m);
        st.m = m;
        st.l = st.l * f0 + ml.y * f1;
#pragma unroll
        for (int nn = 0; nn < 4; nn++)
          st.o[nn] = st.o[nn] * f0 + *(const f32x4 *)&s_o[wave][col * kHeadDim + 16 * nn + 4 * kg] * f1;
        __builtin_amdgcn_wave_barrier();
      }
#pragma unroll
      for (int nn = 0; nn < 4; nn++)
        *(f32x4 *)&s_o[wave][col * kHeadDim + 16 * nn + 4 * kg] = st.o[nn];
      if (kg == 0)
        s_ml[wave][col] = float2{st.m, st.l};
    }
  }
  __syncthreads();
  if (!ok)
    return;
  const int w0 = slot * a.parts;
  for (int i = part * 64 + lane; i < a.G * (kHeadDim / 4); i += a.parts * 64) {
    const int hh = i / (kHeadDim / 4);
    float m = kLowest, l = 0.0f;
    for (int p = 0; p < a.parts; p++)
      m = fmaxf(m, s_ml[w0 + p][hh].x);
    f32x4 o{0.0f, 0.0f, 0.0f, 0.0f};
    for (int p = 0; p < a.parts; p++) {
      const float f = __builtin_amdgcn_exp2f(s_ml[w0 + p][hh].x - m);
      l = fmaf(s_ml[w0 + p][hh].y, f, l);
      o += *(const f32x4 *)&s_o[w0 + p][4 * i] * f;
    }
    if (LAST) {
      put(a.out, (int64_t)b * a.out_stride + (int64_t)g * a.G * kHeadDim + 4 * i,
          o * out_factor(m, l, sink_of(a, g, hh)), a.out_bf16);
    } else {
      const int64_t at = piece_at(s, s.splits + e, b) + g * a.G + hh;
      *(f32x4 *)(s.ws_o + at * kHeadDim + 4 * (i % (kHeadDim / 4))) = o;
      if (i % (kHeadDim / 4) == 0)
        *(float2 *)(s.ws_ml + 2 * at) = float2{m, l};
    }
  }
}

// ---- host side ------------------------------------------------------------------------

constexpr int kSharedWgs = 512;    // workgroups that a prefix launch aims at: two per CU
constexpr int kSharedPieces = 2048; // pieces (times sequences) per kind, at most, or one per sequence
constexpr int kOwnSteps = 72;      // steps of own blocks that one workgroup takes in the last launch

struct SharedPlan {
  int nt, wq, seqs_per_wave;
  int64_t tiles;
  int splits, min_steps, own_pieces;
  size_t o, total; // workspace
};

static SharedPlan shared_plan(int32_t B, int32_t n_groups, int32_t n_q_heads, int32_t n_kv_heads,
                              int32_t max_shared, int32_t max_own, bool blk, bool fine) {
  SharedPlan p{};
  const int G = n_q_heads / n_kv_heads;
  const int64_t avg = n_groups > 0 ? std::max<int64_t>(1, ((int64_t)B + n_groups - 1) / n_groups) : 1;
  const int64_t cols = avg * G;
  p.nt = cols <= 16 ? 1 : cols <= 32 || fine || !blk ? 2 : 4;
  p.seqs_per_wave = 16 * p.nt / G;
  const int64_t wave_tiles = (avg + p.seqs_per_wave - 1) / p.seqs_per_wave;
  p.wq = wave_tiles >= 3 ? 4 : (int)wave_tiles;
  const int64_t per = (int64_t)p.seqs_per_wave * p.wq;
  p.tiles = B / per + n_groups;
  const int64_t busy = n_groups * ((avg + per - 1) / per) * n_kv_heads;
  const int64_t steps = ((int64_t)max_shared + 1) / 2;
  const int wt = kSharedWaves / p.wq;
  p.min_steps = 4 * wt;
  const int64_t room = std::max<int64_t>(1, kSharedPieces / std::max(B, 1));
  int64_t splits = std::min(kSharedWgs / std::max<int64_t>(busy, 1), room);
  splits = std::min(splits, (steps + p.min_steps - 1) / p.min_steps);
  p.splits = n_groups > 0 ? (int)std::max<int64_t>(1, splits) : 0;
  const int64_t own_steps = (((int64_t)max_own + kBlockTokens - 1) / kBlockTokens + 1) / 2;
  p.own_pieces = (int)std::min((own_steps + kOwnSteps - 1) / kOwnSteps - 1, room);
  p.own_pieces = std::max(p.own_pieces, 0);
  if (B > kSharedPieces)
    p.own_pieces = 0;
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  const size_t rows = (size_t)(p.splits + p.own_pieces) * B * n_q_heads;
  p.o = up(rows * 8);
  p.total = p.o + rows * kHeadDim * 4;
  return p;
}

static bool shared_sizes_ok(int32_t B, int32_t n_groups, int32_t n_q_heads, int32_t n_kv_heads,
                            int32_t max_shared, int32_t max_own) {
  return B >= 0 && n_groups >= 0 && n_q_heads > 0 && n_kv_heads > 0 && n_kv_heads <= 8 &&
         n_q_heads % n_kv_heads == 0 && n_q_heads / n_kv_heads <= kHeads && max_shared >= 0 &&
         max_own >= 0;
}

template <bool BLK>
static void launch_prefix(int nt, bool fine, dim3 grid, dim3 block, size_t lds, hipStream_t hs,
                          const SharedArgs &s) {
  if (fine && nt == 1)
    hipLaunchKernelGGL((shared_prefix_kernel<BLK, 1, true>), grid, block, lds, hs, s);
  else if (fine)
    hipLaunchKernelGGL((shared_prefix_kernel<BLK, 2, true>), grid, block, lds, hs, s);
  else if (nt == 1)
    hipLaunchKernelGGL((shared_prefix_kernel<BLK, 1, false>), grid, block, lds, hs, s);
  else if (nt == 2)
    hipLaunchKernelGGL((shared_prefix_kernel<BLK, 2, false>), grid, block, lds, hs, s);
  else if constexpr (BLK)
    hipLaunchKernelGGL((shared_prefix_kernel<BLK, 4, false>), grid, block, lds, hs, s);
}

template <bool LAST>
static void launch_own(bool blk, bool fine, dim3 grid, dim3 block, hipStream_t hs,
                       const SharedArgs &s) {
  if (blk && fine)
    hipLaunchKernelGGL((shared_own_kernel<true, true, LAST>), grid, block, 0, hs, s);
  else if (blk)
    hipLaunchKernelGGL((shared_own_kernel<true, false, LAST>), grid, block, 0, hs, s);
  else if (fine)
    hipLaunchKernelGGL((shared_own_kernel<false, true, LAST>), grid, block, 0, hs, s);
  else
    hipLaunchKernelGGL((shared_own_kernel<false, false, LAST>), grid, block, 0, hs, s);
}

} // namespace gkv

extern "C" size_t gkv_shared_workspace_bytes(int32_t B, int32_t n_groups, int32_t n_q_heads,
                                             int32_t n_kv_heads, int32_t max_shared_blocks,
                                             int32_t max_own) {
  using namespace gkv;
  if (!shared_sizes_ok(B, n_groups, n_q_heads, n_kv_heads, max_shared_blocks, max_own))
    return 0;
  size_t most = 0; // (whatever the formats)
  for (int k = 0; k < 4; k++)
    most = std::max(most, shared_plan(B, n_groups, n_q_heads, n_kv_heads, max_shared_blocks, max_own,
                                      k & 1, k & 2).total);
  return most;
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
  s.seqs_per_wave = p.seqs_per_wave;
  s.wq = p.wq;
  s.splits = p.splits;
  s.min_steps = p.min_steps;
  s.own_pieces = p.own_pieces;
  s.own_steps = kOwnSteps;
  if (B == 0)
    return GKV_OK;
  // waves per (sequence, head): a few steps each, more where few sequences are there
  const int64_t own = std::min<int64_t>((((int64_t)max_own + 15) / 16 + 1) / 2, kOwnSteps);
  a.parts = 1;
  while (a.parts < 8 && ((int64_t)2 * a.parts * B * Hkv <= 2048 || own > 16 * a.parts))
    a.parts *= 2;
  a.heads_per_wg = std::min(8 / a.parts, Hkv);
  const int64_t own_wgs = (int64_t)B * ((Hkv + a.heads_per_wg - 1) / a.heads_per_wg);
  const int own_threads = 64 * a.parts * a.heads_per_wg;
  const int64_t prefix_wgs = p.tiles * p.splits * Hkv;
  if (!grid_fits(own_wgs, own_threads) || !grid_fits(prefix_wgs, 64 * kSharedWaves))
    return GKV_ERR_UNSUPPORTED;
  if (p.total > 0 && (!workspace || workspace_bytes < p.total))
    return GKV_ERR_WORKSPACE;
  s.ws_ml = (float *)workspace;
  s.ws_o = (float *)((char *)workspace + p.o);
  hipStream_t hs = (hipStream_t)stream;
  if (p.splits > 0) {
    const size_t lds = p.wq == kSharedWaves ? 0 : (size_t)kSharedWaves / 2 * p.nt * 5 * 64 * 16;
    const dim3 grid((unsigned)prefix_wgs), block(64 * kSharedWaves);
    if (blk)
      launch_prefix<true>(p.nt, fine, grid, block, lds, hs, s);
    else
      launch_prefix<false>(p.nt, fine, grid, block, lds, hs, s);
    if ((st = launch_status("shared_prefix_kernel")))
      return st;
  }
  const dim3 block(own_threads);
  if (p.own_pieces > 0) {
    launch_own<false>(blk, fine, dim3((unsigned)own_wgs, (unsigned)p.own_pieces), block, hs, s);
    if ((st = launch_status("shared_own_kernel")))
      return st;
  }
  launch_own<true>(blk, fine, dim3((unsigned)own_wgs), block, hs, s);
  return launch_status("shared_own_kernel");
}
