// Causal attention of prompts, or of chunks that continue a cached history, with a
// sliding window and kept first tokens, over bf16 or block-scaled e4m3 caches.
//
// Row j of prompt b is position start + j and sees position t iff t <= start + j
// and (window 0, or t < kept, or t > start + j - window). Positions before start come
// from the cache, the others from the packed bf16 rows. 4 * 64 operations a
// query head, row and position seen, against 256 bytes of K and V that 8 heads
// and 32 rows or more share: bound by the issue of vector and matrix instructions (32
// keys a wave: 57 vector instructions, 16 of them exponentials, about 45 for
// staging, queries and masks, and 8 matrix ops of 32 cycles). Counted for 8 chunks
// after 1536 cached tokens (159 us): vector units busy 57% of the time, matrix units
// 28%, LDS about 45%; what is left is the chain of one wave, which the three others
// of its SIMD do not cover to the end.
//
// Work: one workgroup per (prompt, kv head, block of queries), eight waves (or
// the largest multiple of the group's heads below): wave = (32 queries, query head),
// so with 8 heads a block is 32 queries, with one 256. All waves share the K and V
// tiles (64 keys) in LDS.
//
// Matrix cores, 32x32 output, K = 16, all operands fp16: S^T[key][query] = K Q^T,
// O^T[dim][query] += V^T P^T. K: e4m3 codes and bf16 magnitudes 2^-14 .. 2^16 are
// fp16 values (below, an absolute error of 2^-25; beyond, flagged when staged). q and P
// are rounded to fp16's 11 bits, q after a power of two that brings its row's
// largest element into [1, 2): a score is off by at most 2^-11 sum |q k| / 8, a
// weight by its own rounding, 2^-11, beside it; the bf16 output's is 2^-8
// (q in two bf16 pieces, 16 bits, doubled the first product and spilled: 204 us
// against 172 for 8 chunks of 100 .. 700 rows after 1536 cached ones, before the
// staging was trimmed). V is
// staged as v * 2^-10 (exact for bf16 magnitudes 2^-4 .. 2^26, an absolute error of at
// most 2^-15 below, inf above, which is flagged). A lane (half h, query n)
// holds 16 scores of one query, keys 8 i + 4 h + 0..3 of the 32; these are its
// P^T operand slots if V^T's operand takes the same keys, so V^T is stored in that
// order and P never leaves its lane. The block's K scale goes into the factor of
// the exponent's FMA (a lane's first 8 scores are one block, the others the
// next), the V scale into V^T when it is staged.
//
// Tiles: each wave fetches one 16-key piece of K or V of the next tile into
// registers before the tile's compute (16 to 32 bytes a lane), and converts and
// writes it into the other LDS buffer afterwards: one barrier per tile. K stands
// by keys, V by dimensions, rows of 128 bytes and 16 of padding, so that operand
// reads meet no bank twice. A block's codes are expanded once
// per workgroup. Kept positions' tiles come first, then the window's; blocks that
// no query of the workgroup sees are not read.
//
// Few workgroups (at most one per CU): sixteen waves, two groups of eight that take
// the tiles in turn with LDS buffers of their own and join their sums at the end.
//
// Weights are taken against a reference that moves only when a lane's 16 of a step sum to
// more than 2^15 (or to a NaN); it then goes 8 bits below the largest score met, and the
// weights are formed again. fp16 holds them in 11 bits from 2^-14 to 2^16, so that
// a weight has them down to 2^-22 of a row's largest and is 0 only below 2^-33 of it: a
// first key that takes nearly all the weight leaves the others theirs. (The reference
// starts below every score, not at the sink, which joins at the end in fp32: against a
// sink 18 nats above the scores the weights would all be 0. It costs a row's first step
// a second forming of its weights: 8 chunks after 1536 cached tokens 156 -> 160 us, 12
// prompts with a window of 128 106.5 -> 109. References 10 and 12 bits below the largest score
// move more often: 166 and 174, 111 and 119.)
#include "kept.hpp"
#include "lds_dma.hpp"

#include <algorithm>
#include <climits>

namespace gkv {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kPTile = 64;              // keys per tile
constexpr int kPRow = kPTile + 8;       // 16-bit values per LDS row (a key's dims, a dim's keys)
constexpr int kPQueries = 32;           // queries per wave
constexpr float kPVScale = 0x1p-10f;    // V is staged as fp16 of v * kPVScale
constexpr float kPQScale = 0.125f * kLog2e;
constexpr float kPLowest = -1e30f;      // the weights' reference before any score (log2 units)
constexpr float kPLift = 8.0f;          // bits from the reference up to the largest score, when it moves
constexpr float kPSum = 32768.0f;       // a lane's weights of a step, at most: none reaches fp16's end
// Grids of at most one workgroup per CU get two groups of waves a workgroup: a CU's
// SIMDs then hold four waves, as with two workgroups. Where two fit, a second group only
// takes the other's place, and a single tile cannot be split. Measured (us, one group /
// two, 8 kv heads, codes): one prompt of 32 rows 9.6 / 10.2, of 200 13.3 / 12.8, of 1024
// 38.5 / 32.6; 512 rows after 30000 738 / 591; 8 chunks of up to 128 after 2048 with a
// window of 256 19.8 / 18.5; 416 workgroups (2 of up to 800 after 4096) 171 / 187. How much
// history a chunk has the host does not know: 16 to 64 rows after 16 cached ones 8.6 / 10.0,
// after 128 12.0 / 12.1, after 512 23.2 / 20.6, after 2048 64.6 / 52.3.
constexpr int64_t kPFewWgs = 256;
constexpr int kPShort = 128; // rows of a prompt without a history that stay with one group
constexpr int kPBand = 2;               // query blocks per band of the grid order

struct KeptPrefillArgs {
  const int32_t *cu, *start;
  const float *q;
  int64_t q_stride;
  const float *cos_tab, *sin_tab;
  const char *k, *v;   // packed rows (NULL: every key from the cache)
  int kv_stride;       // bytes per packed row
  const char *kc, *vc; // the paged cache
  const float *scales; // block format (NULL: bf16)
  const int32_t *table;
  int table_stride, num_blocks;
  KeptRow row;
  const float *sinks;
  int B, G, n_kv_heads, subs, kept, window, max_len, n_qblocks, band;
  void *out;
  int64_t out_stride;
  int out_bf16;
  uint32_t *dev_err;
};

// What a wave fetches of a tile: a 16-key piece of K or V.
struct Piece {
  u32x4 x[2];
  float scale; // of codes
  bool hist;   // a block of the cache (else packed rows)
  bool miss;   // ... that is not there, or that nobody sees
  int p;       // its first position
};

// Keeps a uniform branch a branch (its body is not worth running for nothing).
#define GKV_KEEP_BRANCH asm volatile("")

__device__ __forceinline__ uint32_t f16_pair(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), f16x2));
}

// The value of lane (l + N) % 16 within each row of 16 lanes (DPP row_ror).
template <int N>
__device__ __forceinline__ float row_rotate(float x) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x120 + N, 0xf, 0xf, false));
}

// TASKS: pieces a wave fetches of each tile (1 with eight waves, else 2). GROUPS:
// groups of eight waves that take the tiles in turn (2: TASKS is 1).
template <int TASKS, int GROUPS>
__global__ __launch_bounds__(512 * GROUPS) __attribute__((amdgpu_waves_per_eu(TASKS == 1 ? 4 : 2)))
void kept_prefill_kernel(KeptPrefillArgs a) {
  constexpr int D = kHeadDim;
  __shared__ __attribute__((aligned(16))) uint16_t s_kv_all[GROUPS][2][2][kPTile * kPRow]; // [][buffer][K, V]
  __shared__ __attribute__((aligned(16))) uint16_t s_q[8][kPQueries * kPRow]; // a wave's rows: q, then the output
  __shared__ float s_ks_all[GROUPS][2][4]; // K scale of each block of a tile, negative: it is not there

  // Grid order: kv head fastest (the workgroups of a head on one XCD share its
  // K/V in that L2), bands of query blocks longest first, a prompt's blocks of a band
  // together.
  int id = blockIdx.y * kGridRow + blockIdx.x;
  const int g = id % a.n_kv_heads;
  id /= a.n_kv_heads;
  const int band = id / (a.B * a.band), w = id - band * (a.B * a.band);
  const int b = w / a.band;
  const int qb = a.n_qblocks - 1 - (band * a.band + w % a.band);
  if (qb < 0)
    return;
  const int row0 = uniform(a.cu[b]), L = uniform(a.cu[b + 1]) - row0;
  const int qn = kPQueries * a.subs, q0 = qb * qn; // the block's queries
  if (q0 >= L)
    return;
  const int tid = threadIdx.x, lane = tid & 63;
  const int group = GROUPS > 1 ? uniform(tid >> 9) : 0, wave = uniform((tid >> 6) & 7);
  auto &s_kv = s_kv_all[group];
  auto &s_ks = s_ks_all[group];
  const int n = lane & 31, h = lane >> 5;
  int start = a.start ? uniform(a.start[b]) : 0;
  if (start < 0 || start % kBlockTokens != 0) {
    if (tid == 0 && a.dev_err)
      atomicOr(a.dev_err, GKV_DEVERR_ALIGN);
    start = 0; // (the prompt's outputs are then meaningless, but finite)
  }
  // positions a full layer's table row can hold; a prompt that runs past takes its
  // further angles at the last that fits
  const int cap = a.kc && a.row.ring_blocks == 0
                      ? (int)min((int64_t)a.table_stride * kBlockTokens, (int64_t)INT_MAX)
                      : INT_MAX;
  // (the grid covers max_len rows)
  if ((start > cap - L || L > a.max_len) && q0 == 0 && tid == 0 && a.dev_err)
    atomicOr(a.dev_err, GKV_DEVERR_LENGTH);
  if (start > INT_MAX - L)
    start = 0; // (no such positions)
  const int p0 = start + q0, p_last = start + min(q0 + qn, L) - 1;
  const int W = a.window;
  // first position that the window of any query holds; its tile's start
  const int lo = W > 0 ? max(p0 - W + 1, 0) : 0;
  const int k_lo = lo & ~(kPTile - 1);
  const int kept = W > 0 ? a.kept : 0;
  const int n_first = min(kept / kPTile + (kept % kPTile != 0), k_lo / kPTile); // kept positions' tiles
  const int n_tiles = (p_last - k_lo) / kPTile + 1 + n_first;
  auto tile_pos = [&](int t) { return t < n_first ? t * kPTile : k_lo + (t - n_first) * kPTile; };
  const int hist_end = a.k ? start : INT_MAX;
  const int lo_blk = lo / kBlockTokens;
  const int to_ring = kept_entry(a.row, max(lo_blk, a.row.kept_blocks)) - max(lo_blk, a.row.kept_blocks);
  const int ring_end = a.row.kept_blocks + a.row.ring_blocks;
  const int n_waves = a.G * a.subs;

  // Block id of a piece of tile t (kNone: not from the cache, or seen by nobody; outside any pool). It
  // and the scales come through vector loads: a scalar load in flight would
  // hold up the wait for every LDS read behind it.
  constexpr int kNone = -1;
  const __amdgpu_buffer_rsrc_t table_row =
      head_rsrc(a.table + (int64_t)b * a.table_stride, a.table ? 4 * a.table_stride : 0);
  auto id_of = [&](int t, int task) -> int {
    const int p = tile_pos(t) + kBlockTokens * (task & 3);
    if (t >= n_tiles || p >= hist_end || p > p_last)
      return kNone;
    int e = p / kBlockTokens;
    if (W > 0 && e >= a.row.kept_blocks) {
      GKV_KEEP_BRANCH;
      if (e < lo_blk)
        return kNone;
      if (a.row.ring_blocks > 0) { // the blocks seen, at most the ring's, wrap once
        e += to_ring;
        if (e >= ring_end)
          e -= a.row.ring_blocks;
      }
    }
    if (e >= a.table_stride)
      return kNone;
    return __builtin_amdgcn_raw_buffer_load_b32(table_row, 0, 4 * e, 0);
  };
  bool bad = false, range = false;
  // (lane roles: K's piece as (kg, t), V's blocks as (kg, c), V's rows as (kg, d).
  // The lane is made opaque in each use, so that the offsets are formed there and not
  // kept in registers, of which there are none to spare, through the loop.)
  auto opaque_lane = [&]() {
    int x = lane;
    asm volatile("" : "+v"(x));
    return x;
  };
  auto fetch = [&](Piece &x, int t, int task, int id_loaded) {
    const int id = uniform(id_loaded);
    const int ln = opaque_lane(), c16 = ln & 15, kg = ln >> 4;
    const bool is_v = task >= 4;
    x.p = tile_pos(t) + kBlockTokens * (task & 3);
    x.scale = 0.0f;
    x.hist = x.p < hist_end;
    x.miss = false;
    if (x.hist) {
      GKV_KEEP_BRANCH;
      const bool ok = (uint32_t)id < (uint32_t)a.num_blocks;
      if (!ok) { // flagged if id_of read it (its conditions)
        GKV_KEEP_BRANCH;
        const int e = x.p / kBlockTokens;
        bad |= x.p <= p_last && (W == 0 || e < a.row.kept_blocks || e >= lo_blk) &&
               (a.row.ring_blocks > 0 || e < a.table_stride);
      }
      x.miss = !ok;
      const int64_t hb = (int64_t)(ok ? id : 0) * a.n_kv_heads + g;
      const char *src = is_v ? a.vc : a.kc;
      if (a.scales) {
        GKV_KEEP_BRANCH;
        const __amdgpu_buffer_rsrc_t r = head_rsrc(src + hb * 1024, ok ? 1024 : 0);
        x.x[0] = __builtin_amdgcn_raw_buffer_load_b128(r, is_v ? (c16 * 4 + kg) * 16 : ln * 16, 0, 0);
        const __amdgpu_buffer_rsrc_t sr = head_rsrc(a.scales + 2 * hb, ok ? 8 : 0);
        x.scale = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(sr, is_v ? 4 : 0, 0, 0));
      } else {
        const __amdgpu_buffer_rsrc_t r = head_rsrc(src + hb * 2048, ok ? 2048 : 0);
        x.x[0] = __builtin_amdgcn_raw_buffer_load_b128(r, ln * 16, 0, 0);
        x.x[1] = __builtin_amdgcn_raw_buffer_load_b128(r, ln * 16 + 1024, 0, 0);
      }
    } else {
      // packed rows: those past the prompt read as zeros
      const int first = uniform(x.p - start), rows = uniform(max(min(L - first, kBlockTokens), 0));
      const char *src = (is_v ? a.v : a.k) + (int64_t)(row0 + min(first, L - 1)) * a.kv_stride + g * D * 2;
      const __amdgpu_buffer_rsrc_t r = head_rsrc(src, max(rows * a.kv_stride - g * D * 2, 0));
      if (is_v) {
        u32x2 y[4];
#pragma unroll
        for (int i = 0; i < 4; i++)
          y[i] = __builtin_amdgcn_raw_buffer_load_b64(r, (4 * kg + i) * a.kv_stride + c16 * 8, 0, 0);
        x.x[0] = u32x4{y[0][0], y[0][1], y[1][0], y[1][1]};
        x.x[1] = u32x4{y[2][0], y[2][1], y[3][0], y[3][1]};
      } else {
        x.x[0] = __builtin_amdgcn_raw_buffer_load_b128(r, c16 * a.kv_stride + kg * 16, 0, 0);
        x.x[1] = __builtin_amdgcn_raw_buffer_load_b128(r, c16 * a.kv_stride + 64 + kg * 16, 0, 0);
      }
    }
  };
  // Converts a piece and writes it into LDS. K: key rows; V: dimension rows, the
  // tokens of each 16 in the order of the operand slots (8 i + 4 h + r at 8 h + 4 i + r).
  auto store = [&](Piece &x, int buf, int task) {
    const int blk = task & 3, ln = opaque_lane(), c16 = ln & 15, kg = ln >> 4;
    const bool is_v = task >= 4;
    const bool codes = x.hist && a.scales;
    if (x.hist && (x.p < lo || x.p + kBlockTokens - 1 > p_last)) {
      // a cached piece with tokens that no query of the workgroup sees: what they
      // hold, which may be anything, becomes 0
      GKV_KEEP_BRANCH;
      auto seen = [&](int r) {
        const int p = x.p + r;
        return p <= p_last && (p >= lo || p < kept);
      };
      if (!is_v) {
        if (!seen(c16))
          x.x[0] = x.x[1] = u32x4{0, 0, 0, 0};
      } else if (codes) {
        uint32_t keep = 0;
#pragma unroll
        for (int r = 0; r < 4; r++)
          keep |= seen(4 * kg + r) ? 0xffu << (8 * r) : 0u;
        x.x[0] &= u32x4{keep, keep, keep, keep};
      } else {
        const uint32_t m01 = (seen(4 * kg) ? 0xffffu : 0u) | (seen(4 * kg + 1) ? 0xffff0000u : 0u);
        const uint32_t m23 = (seen(4 * kg + 2) ? 0xffffu : 0u) | (seen(4 * kg + 3) ? 0xffff0000u : 0u);
        x.x[0] &= u32x4{m01, m23, m01, m23};
        x.x[1] &= u32x4{m01, m23, m01, m23};
      }
    }
    if (!is_v) {
      u32x4 lo4, hi4;
      if (codes) {
        GKV_KEEP_BRANCH;
        const u32x2 y0 = codes_to_f16(x.x[0][0]), y1 = codes_to_f16(x.x[0][1]);
        const u32x2 y2 = codes_to_f16(x.x[0][2]), y3 = codes_to_f16(x.x[0][3]);
        lo4 = u32x4{y0[0], y0[1], y1[0], y1[1]};
        hi4 = u32x4{y2[0], y2[1], y3[0], y3[1]};
        // a scale that is not finite makes its block NaN, for the rows that see it
        if (!(x.scale < INFINITY)) {
          GKV_KEEP_BRANCH;
          lo4 = hi4 = u32x4{0x7e007e00u, 0x7e007e00u, 0x7e007e00u, 0x7e007e00u};
          x.scale = 1.0f;
        }
      } else {
        GKV_KEEP_BRANCH;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          lo4[i] = f16_pair(__uint_as_float(x.x[0][i] << 16), __uint_as_float(x.x[0][i] & 0xffff0000u));
          hi4[i] = f16_pair(__uint_as_float(x.x[1][i] << 16), __uint_as_float(x.x[1][i] & 0xffff0000u));
        }
        // beyond fp16: a score of -inf would count for nothing without a trace
        typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
        u16x2 top{0, 0};
#pragma unroll
        for (int i = 0; i < 4; i++) {
          top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, lo4[i] & 0x7fff7fffu));
          top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, hi4[i] & 0x7fff7fffu));
        }
        if (__any(((__builtin_bit_cast(uint32_t, top) + 0x04000400u) & 0x80008000u) != 0))
          range = true;
      }
      uint16_t *dst = s_kv[buf][0] + (kBlockTokens * blk + c16) * kPRow + 8 * kg;
      *(u32x4 *)dst = lo4;
      *(u32x4 *)(dst + 32) = hi4;
      if (ln == 0) {
        s_ks[buf][blk] = x.miss ? -1.0f : codes ? x.scale : 1.0f;
      }
      return;
    }
    // tokens 4kg .. 4kg+3 of dimension d at dst + d rows
    uint16_t *dst = s_kv[buf][1] + 16 * blk + 8 * (kg & 1) + 4 * (kg >> 1);
    if (codes) {
      GKV_KEEP_BRANCH;
      dst += c16 * kPRow;
      const float s = __uint_as_float(uniform(__float_as_uint(x.scale * kPVScale)));
      if ((__float_as_uint(s) & 0x7fffffu) == 0) {
        // a power of two: the conversion applies it
        GKV_KEEP_BRANCH;
#pragma unroll
        for (int nn = 0; nn < 4; nn++)
          *(u32x2 *)(dst + 16 * nn * kPRow) = codes_to_f16(x.x[0][nn], s);
      } else {
        GKV_KEEP_BRANCH;
#pragma unroll
        for (int nn = 0; nn < 4; nn++) {
          const f32x2 f0 = __builtin_amdgcn_cvt_pk_f32_fp8((int)x.x[0][nn], false);
          const f32x2 f1 = __builtin_amdgcn_cvt_pk_f32_fp8((int)x.x[0][nn], true);
          *(u32x2 *)(dst + 16 * nn * kPRow) = u32x2{f16_pair(f0[0] * s, f0[1] * s), f16_pair(f1[0] * s, f1[1] * s)};
        }
      }
    } else if (x.hist) {
      GKV_KEEP_BRANCH;
      dst += c16 * kPRow;
#pragma unroll
      for (int nn = 0; nn < 4; nn++) { // dims c + 32 (nn / 2) + 16 (nn % 2)
        const uint32_t t01 = x.x[nn / 2][2 * (nn & 1)], t23 = x.x[nn / 2][2 * (nn & 1) + 1];
        *(u32x2 *)(dst + 16 * nn * kPRow) =
            u32x2{f16_pair(__uint_as_float(t01 << 16) * kPVScale, __uint_as_float(t01 & 0xffff0000u) * kPVScale),
                  f16_pair(__uint_as_float(t23 << 16) * kPVScale, __uint_as_float(t23 & 0xffff0000u) * kPVScale)};
      }
    } else {
      // rows 4kg + i, dims 4 c .. 4 c + 3: 4 x 4 turned
      GKV_KEEP_BRANCH;
      dst += 4 * c16 * kPRow;
#pragma unroll
      for (int d = 0; d < 4; d++) {
        float f[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const uint32_t y = x.x[i / 2][2 * (i & 1) + d / 2];
          f[i] = __uint_as_float(d & 1 ? y & 0xffff0000u : y << 16) * kPVScale;
        }
        *(u32x2 *)(dst + d * kPRow) = u32x2{f16_pair(f[0], f[1]), f16_pair(f[2], f[3])};
      }
    }
  };

  Piece pc[TASKS];
  int ids[TASKS];
  int ids0[TASKS];
#pragma unroll
  for (int i = 0; i < TASKS; i++) {
    const int task = wave + i * n_waves;
    ids0[i] = ids[i] = kNone;
    if (task < 8) {
      ids0[i] = id_of(group, task);
      ids[i] = id_of(group + GROUPS, task);
    }
  }

  // ---- the queries ----
  // Read by whole rows: lane (r, c) = (lane / 16, lane % 16) holds dims 4 c .. 4 c + 3 of
  // rows 4 i + r, and lane c ^ 8 of its 16 the other half of their RoPE pairs. Rotated,
  // scaled and rounded they go through LDS (the wave's own rows) into the operands'
  // order. (Operand order straight from memory reads 32 bytes of 32 rows an
  // instruction: lines left L1 before their rest was read.)
  const int sub = wave / a.G, head = g * a.G + wave % a.G;
  const int p0s = p0 + kPQueries * sub;             // this wave's queries
  const int p_last_s = min(p0s + kPQueries - 1, start + L - 1);
  const bool active = p0s <= p_last_s;
  uint16_t *sq = s_q[wave];
  f16x8 qv[4];
  float qf; // what the scores of this lane's query are to be multiplied with
  {
    const int r4 = lane >> 4, c = lane & 15;
    constexpr int kRows = 8 / GROUPS; // quads of rows (the groups share a wave's rows)
    const int i0 = kRows * group;
    f32x4 y[kRows], cs[kRows], sn[kRows];
#pragma unroll
    for (int i = 0; i < kRows; i++) {
      const int j = min(q0 + kPQueries * sub + 4 * (i0 + i) + r4, L - 1);
      y[i] = *(const f32x4 *)(a.q + (int64_t)(row0 + j) * a.q_stride + head * D + 4 * c);
      if (a.cos_tab) {
        const int64_t at = (int64_t)min(start + j, cap - 1) * (D / 2) + 4 * (c & 7);
        cs[i] = *(const f32x4 *)(a.cos_tab + at);
        sn[i] = *(const f32x4 *)(a.sin_tab + at);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    // the first pieces, whose addresses wait for the block ids, behind these loads
#pragma unroll
    for (int i = 0; i < TASKS; i++)
      if (wave + i * n_waves < 8)
        fetch(pc[i], group, wave + i * n_waves, ids0[i]);
    __builtin_amdgcn_sched_barrier(0);
    if (a.cos_tab) {
      // x cos -/+ other sin: the sine's sign bit is flipped below c = 8, so that both
      // halves run the same instructions (and round as rope_first and rope_second do)
      const uint32_t flip = c < 8 ? 0x80000000u : 0u;
#pragma unroll
      for (int i = 0; i < kRows; i++)
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const float x = y[i][k], sine = __uint_as_float(__float_as_uint(sn[i][k]) ^ flip);
          y[i][k] = rope_second(swap8(x), x, cs[i][k], sine);
        }
    }
#pragma unroll
    for (int i = 0; i < kRows; i++) {
      float mx = 0.0f;
#pragma unroll
      for (int k = 0; k < 4; k++)
        mx = fmaxf(mx, fabsf(y[i][k]));
      // the row's largest element, over its 16 lanes
      mx = fmaxf(mx, swap8(mx));
      mx = fmaxf(mx, row_rotate<4>(mx));
      mx = fmaxf(mx, row_rotate<2>(mx));
      mx = fmaxf(mx, row_rotate<1>(mx));
      // q * 2^-e, its largest element in [1, 2)
      const int e = min(max((int)(__float_as_uint(mx) >> 23), 27), 227);
      const float down = __uint_as_float((uint32_t)(254 - e) << 23);
      *(u32x2 *)(sq + (4 * (i0 + i) + r4) * kPRow + 4 * c) =
          u32x2{f16_pair(y[i][0] * down, y[i][1] * down), f16_pair(y[i][2] * down, y[i][3] * down)};
      if (c == 0)
        *(float *)(sq + (4 * (i0 + i) + r4) * kPRow + D) =
            kPQScale * __uint_as_float((uint32_t)e << 23); // (in the row's padding)
    }
    if (GROUPS > 1)
      lds_barrier();
    else
      __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int kk = 0; kk < 4; kk++)
      qv[kk] = *(const f16x8 *)(sq + n * kPRow + 8 * h + 16 * kk);
    qf = *(const float *)(sq + n * kPRow + D);
  }
  const int operand = n * kPRow + 8 * h; // this lane's place in an operand's rows
  const float sink2 = a.sinks && active ? a.sinks[head] * kLog2e : -INFINITY;
  float m = kPLowest, l = 0.0f;
  f32x16 o[2];
#pragma unroll
  for (int i = 0; i < 16; i++)
    o[0][i] = o[1][i] = 0.0f;

#pragma unroll
  for (int i = 0; i < TASKS; i++)
    if (wave + i * n_waves < 8)
      store(pc[i], 0, wave + i * n_waves);
  lds_barrier();

  // steps (32 keys from kb on) that this wave's queries see something of: kb in
  // [key_begin, key_end] or below kept; up to window_end some query has left them behind
  const int key_end = active ? p_last_s : -1, key_begin = W > 0 ? max(p0s - W, INT_MIN + 30) - 30 : INT_MIN;
  const int window_end = W > 0 ? p_last_s - W : INT_MIN;
  for (int t = group, buf = 0; t - group < n_tiles; t += GROUPS, buf ^= 1) {
#pragma unroll
    for (int i = 0; i < TASKS; i++) {
      const int task = wave + i * n_waves;
      if (task < 8 && t + GROUPS < n_tiles) {
        fetch(pc[i], t + GROUPS, task, ids[i]);
        ids[i] = id_of(t + 2 * GROUPS, task);
      }
    }
    __builtin_amdgcn_sched_barrier(0); // (the loads stay in front of the compute)
    const int kt = tile_pos(t);
#pragma unroll
    for (int s = 0; s < 2; s++) {
      const int kb = kt + 32 * s;
      if ((GROUPS > 1 && t >= n_tiles) || kb > key_end || (kb < key_begin && kb >= kept))
        continue; // nothing of the step is seen
      f32x16 acc;
#pragma unroll
      for (int i = 0; i < 16; i++)
        acc[i] = 0.0f;
      // a wave in its step goes before those that stage (8 chunks after 1536 cached
      // tokens 162 -> 156 us)
      __builtin_amdgcn_s_setprio(1);
      const uint16_t *krow = s_kv[buf][0] + 32 * s * kPRow + operand;
#pragma unroll
      for (int kk = 0; kk < 4; kk++) {
        const f16x8 kop = *(const f16x8 *)(krow + 16 * kk);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kop, qv[kk], acc, 0, 0, 0);
      }
      const float c0 = qf * s_ks[buf][2 * s], c1 = qf * s_ks[buf][2 * s + 1];
      const bool gone = __any(fminf(c0, c1) < 0.0f);
      if (kb > p0s - 31 || (kb <= window_end && kb + 31 >= kept) || gone) {
        GKV_KEEP_BRANCH;
        // a missing block's tokens count for nothing (their V is 0)
#pragma unroll
        for (int j = 0; j < 2; j++)
          if ((j ? c1 : c0) < 0.0f) {
#pragma unroll
            for (int i = 0; i < 8; i++)
              acc[8 * j + i] = -INFINITY;
          }
        // key kb + 4 h + off is seen iff 0 <= last - off < W, or it is a kept one
        const int ln = opaque_lane(), h = ln >> 5, last = p0s + (ln & 31) - kb - 4 * h;
        const uint32_t wide = W > 0 ? (uint32_t)W : 0x80000000u;
        const int in_kept = kept - kb - 4 * h;
        if (kb < kept) {
#pragma unroll
          for (int i = 0; i < 16; i++) {
            const int off = 8 * (i / 4) + i % 4;
            const bool in = (off <= last) & (((uint32_t)(last - off) < wide) | (off < in_kept));
            acc[i] = in ? acc[i] : -INFINITY;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16; i++)
            acc[i] = (uint32_t)(last - (8 * (i / 4) + i % 4)) < wide ? acc[i] : -INFINITY;
        }
      }
      // (a scale of 0 must not turn a masked score's -inf into a NaN)
      const float d0 = fmaxf(c0, 1e-37f), d1 = fmaxf(c1, 1e-37f);
      f16x8 p[2];
      float sum;
      auto weights = [&](float ref) {
        uint32_t x[8];
        sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const float d = i < 4 ? d0 : d1;
          x[i] = f16_pair(__builtin_amdgcn_exp2f(fmaf(acc[2 * i], d, -ref)),
                          __builtin_amdgcn_exp2f(fmaf(acc[2 * i + 1], d, -ref)));
          sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, x[i]),
                                       f16x2{(_Float16)1.0f, (_Float16)1.0f}, sum, false);
        }
        p[0] = __builtin_bit_cast(f16x8, u32x4{x[0], x[1], x[2], x[3]});
        p[1] = __builtin_bit_cast(f16x8, u32x4{x[4], x[5], x[6], x[7]});
      };
      weights(m);
      if (__any(!(sum <= kPSum))) {
        float m0 = acc[0], m1 = acc[8];
#pragma unroll
        for (int i = 1; i < 8; i++) {
          m0 = fmaxf(m0, acc[i]);
          m1 = fmaxf(m1, acc[8 + i]);
        }
        float mx = fmaxf(m0 * d0, m1 * d1);
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float mn = fmaxf(m, mx - kPLift);
        const float f = __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= f;
#pragma unroll
        for (int i = 0; i < 16; i++) {
          o[0][i] *= f;
          o[1][i] *= f;
        }
        weights(m);
      }
      l += sum;
#pragma unroll
      for (int dt = 0; dt < 2; dt++) {
        const uint16_t *vrow = s_kv[buf][1] + 32 * dt * kPRow + 32 * s + operand;
#pragma unroll
        for (int ks = 0; ks < 2; ks++) {
          const f16x8 vop = *(const f16x8 *)(vrow + 16 * ks);
          o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vop, p[ks], o[dt], 0, 0, 0);
        }
      }
      __builtin_amdgcn_s_setprio(0);
    }
    if (t - group + GROUPS < n_tiles) { // (the same for both groups)
#pragma unroll
      for (int i = 0; i < TASKS; i++)
        if (wave + i * n_waves < 8 && t + GROUPS < n_tiles)
          store(pc[i], buf ^ 1, wave + i * n_waves);
      lds_barrier();
    }
  }
  if (a.dev_err) {
    if ((bad || range) && lane == 0)
      atomicOr(a.dev_err, (bad ? GKV_DEVERR_BLOCK_ID : 0u) | (range ? GKV_DEVERR_RANGE : 0u));
  }

  if (GROUPS > 1) {
    // the second group's sums to the first, through the tiles' place
    static_assert(GROUPS == 1 || 8 * 34 * 64 * 4 <= sizeof(s_kv_all), "a group's sums fit");
    float *sums = (float *)s_kv_all + wave * 34 * 64 + lane;
    lds_barrier();
    if (group == 1) {
      sums[0] = m;
      sums[64] = l;
#pragma unroll
      for (int i = 0; i < 16; i++) {
        sums[64 * (2 + i)] = o[0][i];
        sums[64 * (18 + i)] = o[1][i];
      }
    }
    lds_barrier();
    if (group == 1)
      return;
    const float m1 = sums[0], mm = fmaxf(m, m1);
    const float f0 = __builtin_amdgcn_exp2f(m - mm), f1 = __builtin_amdgcn_exp2f(m1 - mm);
    m = mm;
    l = fmaf(sums[64], f1, l * f0);
#pragma unroll
    for (int i = 0; i < 16; i++) {
      o[0][i] = fmaf(sums[64 * (2 + i)], f1, o[0][i] * f0);
      o[1][i] = fmaf(sums[64 * (18 + i)], f1, o[1][i] * f0);
    }
  }

  // out = o / (l + sink's weight) / kPVScale; 0 for a row that saw nothing
  const int ln = opaque_lane(), n_o = ln & 31, h_o = ln >> 5;
  l += __shfl_xor(l, 32);
  const float M = fmaxf(m, sink2);
  const float f = __builtin_amdgcn_exp2f(m - M);
  const float den = fmaf(l, f, __builtin_amdgcn_exp2f(sink2 - M));
  const float scale = den == 0.0f ? 0.0f : f / den / kPVScale;
  const int q_first = q0 + kPQueries * sub; // this wave's first row of the prompt
  if (a.dev_err) {
    // an output that is not finite, as K and V beyond fp16 give it
    float z = scale * 0.0f;
#pragma unroll
    for (int i = 0; i < 16; i++)
      z = fmaf(o[0][i], 0.0f, fmaf(o[1][i], 0.0f, z));
    if (__any(!(z == 0.0f) && active && q_first + n_o < L) && ln == 0)
      atomicOr(a.dev_err, GKV_DEVERR_RANGE);
  }
  if (!a.out_bf16) {
    if (!active || q_first + n_o >= L)
      return;
    float *dst = (float *)a.out + (int64_t)(row0 + q_first + n_o) * a.out_stride + head * D + 4 * h_o;
#pragma unroll
    for (int dt = 0; dt < 2; dt++)
#pragma unroll
      for (int i = 0; i < 4; i++)
        *(f32x4 *)(dst + 32 * dt + 8 * i) =
            f32x4{o[dt][4 * i], o[dt][4 * i + 1], o[dt][4 * i + 2], o[dt][4 * i + 3]} * scale;
    return;
  }
  // bf16: through LDS (the wave's own rows), so that a row's 128 bytes leave together
  uint16_t *so = sq;
#pragma unroll
  for (int dt = 0; dt < 2; dt++)
#pragma unroll
    for (int i = 0; i < 4; i++) { // dims 32 dt + 8 i + 4 h + 0..3
      const u32x2 y{f32x2_to_bf16_rne(o[dt][4 * i] * scale, o[dt][4 * i + 1] * scale),
                    f32x2_to_bf16_rne(o[dt][4 * i + 2] * scale, o[dt][4 * i + 3] * scale)};
      *(u32x2 *)(so + n_o * kPRow + 32 * dt + 8 * i + 4 * h_o) = y;
    }
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int r = 8 * i + (ln >> 3), slot = ln & 7;
    const u32x4 y = *(const u32x4 *)(so + r * kPRow + slot * 8);
    if (active && q_first + r < L)
      *(u32x4 *)((uint16_t *)a.out + (int64_t)(row0 + q_first + r) * a.out_stride + head * D + slot * 8) = y;
  }
}

} // namespace gkv

extern "C" int gkv_kept_prefill(void *stream, int32_t B, const int32_t *cu_seqlens,
                                const int32_t *start_pos, int32_t max_len, int32_t n_q_heads,
                                const float *q, int64_t q_stride, const float *cos_tab,
                                const float *sin_tab, const void *k, const void *v,
                                gkv_cache_view cache, int32_t kept, int32_t window,
                                const float *sinks, void *out, int64_t out_stride,
                                int32_t out_dtype, uint32_t *dev_err) {
  using namespace gkv;
  if (B < 0 || max_len < 0 || n_q_heads <= 0 || (out_dtype != GKV_F32 && out_dtype != GKV_BF16))
    return GKV_ERR_ARG;
  const bool cached = cache.k != nullptr;
  int st = kept_check(cache, kept, window, cached);
  if (st != GKV_OK)
    return st;
  if (B > 0 && (!cu_seqlens || !q || !out))
    return GKV_ERR_ARG;
  if (n_q_heads % cache.n_kv_heads != 0 || (cos_tab == nullptr) != (sin_tab == nullptr) ||
      (k == nullptr) != (v == nullptr))
    return GKV_ERR_ARG;
  if ((!k && !cached) || (start_pos && !cached) || (cached && cache.ring > 0 && !k))
    return GKV_ERR_ARG; // keys from nowhere; a history needs the cache; a ring holds the history only
  const int G = n_q_heads / cache.n_kv_heads;
  if (G > 8 || cache.n_kv_heads >= (1 << 20))
    return GKV_ERR_UNSUPPORTED; // (16 packed rows take less than 2^31 bytes)
  if (q_stride < (int64_t)n_q_heads * kHeadDim || out_stride < (int64_t)n_q_heads * kHeadDim ||
      q_stride % 4 != 0 || out_stride % (out_dtype == GKV_BF16 ? 8 : 4) != 0)
    return GKV_ERR_ARG;
  if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)q | (uintptr_t)cos_tab | (uintptr_t)sin_tab |
       (uintptr_t)out) % 16 != 0)
    return GKV_ERR_ARG; // 16-byte loads and stores
  KeptPrefillArgs a{};
  a.subs = 8 / G;
  const int qn = kPQueries * a.subs;
  a.n_qblocks = (int)(((int64_t)max_len + qn - 1) / qn);
  a.band = std::min(kPBand, std::max(a.n_qblocks, 1));
  const int64_t grid = (int64_t)((a.n_qblocks + a.band - 1) / a.band) * a.band * B * cache.n_kv_heads;
  if (grid == 0)
    return GKV_OK;
  if (grid >= INT_MAX)
    return GKV_ERR_ARG;
  a.cu = cu_seqlens;
  a.start = start_pos;
  a.q = q;
  a.q_stride = q_stride;
  a.cos_tab = cos_tab;
  a.sin_tab = sin_tab;
  a.k = (const char *)k;
  a.v = (const char *)v;
  a.kv_stride = cache.n_kv_heads * kHeadDim * 2;
  if (cached) {
    a.kc = (const char *)cache.k;
    a.vc = (const char *)cache.v;
    a.scales = cache.v_format == GKV_KV_FP8_BLOCK ? (const float *)cache.v_scale : nullptr;
    a.table = cache.block_table;
    a.table_stride = cache.table_stride;
    a.num_blocks = cache.num_blocks;
    a.row.ring_blocks = cache.ring / kBlockTokens;
  }
  a.row.kept_blocks = kept / kBlockTokens;
  a.sinks = sinks;
  a.B = B;
  a.G = G;
  a.n_kv_heads = cache.n_kv_heads;
  a.kept = kept;
  a.window = window;
  a.max_len = max_len;
  a.out = out;
  a.out_stride = out_stride;
  a.out_bf16 = out_dtype == GKV_BF16;
  a.dev_err = dev_err;
  const dim3 block(64 * G * a.subs);
  const dim3 rows((unsigned)std::min<int64_t>(grid, kGridRow), (unsigned)((grid + kGridRow - 1) / kGridRow));
  if (G * a.subs == 8 && grid <= kPFewWgs && (start_pos || max_len > kPShort))
    hipLaunchKernelGGL((kept_prefill_kernel<1, 2>), rows, dim3(1024), 0, (hipStream_t)stream, a);
  else if (G * a.subs == 8)
    hipLaunchKernelGGL((kept_prefill_kernel<1, 1>), rows, block, 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL((kept_prefill_kernel<2, 1>), rows, block, 0, (hipStream_t)stream, a);
  return launch_status("kept_prefill_kernel");
}
