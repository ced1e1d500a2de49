// Block tables kept on the GPU: blocks taken and given back by the sequences' lengths, rows
// that follow the chosen parents, and the map of new rows to slots.
//
// The state is the table, the lengths and, per block, how many table entries hold it (0: free);
// a length says which entries a row holds (ceil(len / 16)). Blocks are shared freely by a
// reorder; a row that goes on inside a block that others hold gets one of its own from the next
// resize, which names the copy.
//
// The n-th block that a call takes is the n-th lowest free id: that needs no list of
// free blocks, whose order would depend on who gave back first, and keeps the pool's low end dense.
// All of it is whole numbers and sums, so results do not depend on the order of the atomics.
// Everything here moves kilobytes: latency bounds it, and launches and dependent loads are
// what is counted. Of a launch's time 2.5 us are its own and some 1.5 each load that
// waits for another.
#include "gkv_device.hpp"

#include <algorithm>

namespace gkv {

constexpr int kTableThreads = 1024;

struct TablesArgs {
  int32_t *table, *lens, *refs;
  int stride, n_seqs, num_blocks;
  uint32_t *dev_err;
};

__device__ __forceinline__ void flag(uint32_t *dev_err, uint32_t bit) {
  if (dev_err)
    atomicOr(dev_err, bit);
}

__device__ __forceinline__ int blocks_of(int len) { return (int)(((uint32_t)len + 15u) / 16u); }

// A row's length as far as its row goes (a length that no row can have counts as 0).
__device__ __forceinline__ int sane(int len, int stride) {
  return len < 0 || blocks_of(len) > stride ? 0 : len;
}

// ---- init ---------------------------------------------------------------------------

__global__ __launch_bounds__(256) void tables_init_kernel(TablesArgs a) {
  const int64_t n = (int64_t)a.n_seqs * a.stride, step = (int64_t)gridDim.x * 256;
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  for (int64_t i = t; i < n; i += step)
    a.table[i] = -1;
  for (int64_t i = t; i < a.n_seqs; i += step)
    a.lens[i] = 0;
  for (int64_t i = t; i < a.num_blocks; i += step)
    a.refs[i] = 0;
}

// ---- resize ---------------------------------------------------------------------------

struct ResizeArgs {
  TablesArgs t;
  const int32_t *new_lens;
  int32_t *copy_src, *copy_dst;
  int max_rows;
  int32_t *cu_rows, *row_seq, *row_pos;
  int64_t *row_slot;
  int maps, alone; // the rows are asked for; the plan's workgroup carries it out
  // left by the plan for the second launch
  int32_t *ok;    // 1: the call is carried out
  int32_t *old;   // [n_seqs] lengths before the call; -1: the row is left as it is
  int32_t *first; // [n_seqs] place of its first taken block among all; bit 31: that one replaces
                  // the partly filled block that others hold
  int32_t *cu;    // [n_seqs + 1] new rows before each sequence
  int32_t *ids;   // [num_blocks] the blocks taken
};

// Sum over the workgroup of the values before this thread's, and of all.
__device__ __forceinline__ uint64_t scan_before(uint64_t x, uint64_t *s_wave, uint64_t &total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint64_t incl = x;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint64_t v = __shfl_up(incl, off, 64);
    if (lane >= off)
      incl += v;
  }
  __syncthreads(); // (s_wave may still be read for the scan before)
  if (lane == 63)
    s_wave[wave] = incl;
  __syncthreads();
  uint64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kTableThreads / 64; w++) {
    const uint64_t v = s_wave[w];
    before += w < wave ? v : 0;
    total += v;
  }
  return before + incl - x;
}

// What a resize does to one row.
struct RowPlan {
  int old;     // -1: it is left as it is
  bool split;  // the block at its end is held by others too
  int take, rows;
};

__device__ __forceinline__ RowPlan row_plan(const ResizeArgs &a, int s, int len, int want) {
  const TablesArgs &t = a.t;
  RowPlan p{sane(len, t.stride), false, 0, 0};
  if (p.old != len || want < 0 || blocks_of(want) > t.stride) {
    flag(t.dev_err, GKV_DEVERR_LENGTH);
    p.old = -1;
    return p;
  }
  if (want > p.old) {
    if (p.old % kBlockTokens != 0) {
      const int id = t.table[(int64_t)s * t.stride + p.old / kBlockTokens];
      p.split = (uint32_t)id < (uint32_t)t.num_blocks && t.refs[id] > 1;
    }
    p.take = (p.split ? 1 : 0) + blocks_of(want) - blocks_of(p.old);
    p.rows = want - p.old;
  }
  return p;
}

// The sequence that new row r belongs to: the last s with cu[s] <= r, in 0 .. n - 1.
__device__ __forceinline__ int sequence_of(const int32_t *cu, int n, int r) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (int)(((uint32_t)lo + (uint32_t)hi) / 2);
    if (cu[mid] <= r)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// A wave carries out what is planned for sequence s: its entries, their holders and its copy.
__device__ __forceinline__ void apply_sequence(const ResizeArgs &a, int s, bool ok) {
  const TablesArgs &t = a.t;
  const int lane = threadIdx.x & 63;
  int src = 0, dst = 0;
  const int old = a.old[s], taken = a.first[s];
  if (ok && old >= 0) {
    int32_t *row = t.table + (int64_t)s * t.stride;
    const int have = blocks_of(old), want = blocks_of(a.new_lens[s]);
    int at = taken & 0x7fffffff;
    if (taken < 0) {
      if (lane == 0) {
        src = row[have - 1];
        dst = a.ids[at];
        row[have - 1] = dst;
        atomicSub(t.refs + src, 1);
        t.refs[dst] = 1;
      }
      at++;
    }
    for (int j = have + lane; j < want; j += 64) {
      const int id = a.ids[at + j - have];
      row[j] = id;
      t.refs[id] = 1;
    }
    for (int j = want + lane; j < have; j += 64) {
      const int id = row[j];
      row[j] = -1;
      if ((uint32_t)id < (uint32_t)t.num_blocks)
        atomicSub(t.refs + id, 1);
      else
        flag(t.dev_err, GKV_DEVERR_BLOCK_ID);
    }
  }
  if (lane == 0 && a.copy_src) {
    a.copy_src[s] = src;
    a.copy_dst[s] = dst;
  }
}

// A thread maps new row r to its sequence, position and slot.
__device__ __forceinline__ void apply_row(const ResizeArgs &a, int r) {
  const TablesArgs &t = a.t;
  const int s = sequence_of(a.cu, t.n_seqs, r);
  const int old = a.old[s], pos = old + r - a.cu[s];
  if (a.row_seq)
    a.row_seq[r] = s;
  if (a.row_pos)
    a.row_pos[r] = pos;
  if (a.row_slot) {
    // (from the plan alone: the table is being changed; a block that others hold is replaced)
    const int have = blocks_of(old), j = pos / kBlockTokens, taken = a.first[s];
    const int at = taken & 0x7fffffff;
    int id;
    if (j >= have)
      id = a.ids[at + (taken < 0 ? 1 : 0) + j - have];
    else
      id = taken < 0 ? a.ids[at] : t.table[(int64_t)s * t.stride + j];
    a.row_slot[r] = (int64_t)id * kBlockTokens + pos % kBlockTokens;
  }
}

// One workgroup: what each row takes, where its rows begin, and the ids of the blocks; the
// lengths, if there is room for all. A chain of dependent loads (lengths, the block at a row's
// end, its holders), so the holders among which free ids are looked for are
// loaded ahead of it, and of every next round ahead of the scan. With few sequences and rows
// (alone) it carries the plan out itself: a launch less (4 chats by 8 tokens 9.9 us a call with two
// launches, 7 so). 1024 sequences by a token 8.1 us, and 3.7 for the second launch; 512 prompts
// of up to 512 tokens 6 and 3.4.
constexpr int kRefsEach = 16; // holders a thread looks at in one go
__device__ __forceinline__ uint32_t free_mask(const TablesArgs &t, int64_t base) {
  uint32_t free = 0;
  if (base + kRefsEach <= t.num_blocks && ((uintptr_t)t.refs & 15) == 0) {
    int4 x[kRefsEach / 4];
#pragma unroll
    for (int i = 0; i < kRefsEach / 4; i++)
      x[i] = *((const int4 *)(t.refs + base) + i);
#pragma unroll
    for (int i = 0; i < kRefsEach / 4; i++)
      free |= ((x[i].x == 0) | (x[i].y == 0) << 1 | (x[i].z == 0) << 2 | (x[i].w == 0) << 3) << (4 * i);
  } else {
#pragma unroll
    for (int i = 0; i < kRefsEach; i++)
      if (base + i < t.num_blocks && t.refs[base + i] == 0)
        free |= 1u << i;
  }
  return free;
}

__global__ __launch_bounds__(kTableThreads) void tables_plan_kernel(ResizeArgs a) {
  __shared__ uint64_t s_wave[kTableThreads / 64];
  const TablesArgs &t = a.t;
  const int tid = threadIdx.x;
  uint32_t free = free_mask(t, (int64_t)tid * kRefsEach);
  int64_t need = 0, rows = 0;
  int want = 0, row = 0;
  RowPlan p{-1, false, 0, 0};
  for (int s0 = 0; s0 < t.n_seqs; s0 += kTableThreads) {
    const int s = s0 + tid;
    p = RowPlan{-1, false, 0, 0};
    if (s < t.n_seqs) {
      want = a.new_lens[s];
      p = row_plan(a, s, t.lens[s], want);
    }
    uint64_t all; // rows above, blocks below: a thousand rows' sums are under 2^32
    const uint64_t at = scan_before((uint64_t)p.rows << 32 | (uint32_t)p.take, s_wave, all);
    row = (int)(rows + (int64_t)(at >> 32));
    if (s < t.n_seqs) {
      a.old[s] = p.old;
      a.first[s] = (int)((need + (int64_t)(uint32_t)at) & 0x7fffffff) | (p.split ? (int)0x80000000u : 0);
      a.cu[s] = row;
    }
    need += (int64_t)(uint32_t)all;
    rows += (int64_t)(all >> 32);
  }
  bool ok = need <= t.num_blocks && rows <= a.max_rows;
  // the lowest free ids, as many as are needed
  int64_t found = 0;
  constexpr int64_t kRound = (int64_t)kTableThreads * kRefsEach;
  for (int64_t r0 = 0; ok && found < need && r0 < t.num_blocks; r0 += kRound) {
    const int64_t base = r0 + (int64_t)tid * kRefsEach;
    const uint32_t next = free_mask(t, base + kRound);
    uint64_t all;
    int64_t at = found + (int64_t)scan_before(__popc(free), s_wave, all);
    for (; free != 0 && at < need; free &= free - 1)
      a.ids[at++] = (int)base + __ffs(free) - 1;
    found += (int64_t)all;
    free = next;
  }
  ok = ok && found >= need;
  if (tid == 0) {
    *a.ok = ok;
    a.cu[t.n_seqs] = (int)rows;
    if (a.cu_rows)
      a.cu_rows[t.n_seqs] = ok ? (int)rows : 0;
    if (!ok)
      flag(t.dev_err, GKV_DEVERR_CAPACITY);
  }
  if (t.n_seqs <= kTableThreads) { // (all is still at hand)
    if (tid < t.n_seqs) {
      if (ok && p.old >= 0)
        t.lens[tid] = want;
      if (a.cu_rows)
        a.cu_rows[tid] = ok ? row : 0;
    }
    if (a.alone) {
      __syncthreads();
      for (int s = tid >> 6; s < t.n_seqs; s += kTableThreads / 64)
        apply_sequence(a, s, ok);
      for (int r = tid; ok && r < (a.maps ? (int)rows : 0); r += kTableThreads)
        apply_row(a, r);
    }
    return;
  }
  __syncthreads();
  for (int s = tid; s < t.n_seqs; s += kTableThreads) {
    if (a.cu_rows)
      a.cu_rows[s] = ok ? a.cu[s] : 0;
    if (ok && a.old[s] >= 0)
      t.lens[s] = a.new_lens[s];
  }
}

// A wave per sequence; behind those, a thread per new row.
__global__ __launch_bounds__(256) void tables_apply_kernel(ResizeArgs a, int seq_wgs) {
  const bool ok = *a.ok != 0;
  if ((int)blockIdx.x < seq_wgs) {
    const int s = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (s < a.t.n_seqs)
      apply_sequence(a, s, ok);
    return;
  }
  const int64_t r = (int64_t)((int)blockIdx.x - seq_wgs) * 256 + threadIdx.x;
  if (ok && r < a.cu[a.t.n_seqs])
    apply_row(a, (int)r);
}

// ---- reorder ----------------------------------------------------------------------------

struct ReorderArgs {
  TablesArgs t;
  const int32_t *parents;
  int per;             // rows of a group
  int width_log;       // columns of a tile: 2^width_log
  int tiles;           // tiles per group that have a workgroup of their own (1: one takes all)
  int32_t *shared;     // NULL, or per group the leading blocks that all its rows hold
};

// A group's parents (places in the group, -1: none) and lengths into LDS; the most
// blocks that one of its rows holds.
__device__ __forceinline__ int load_group(const ReorderArgs &a, int base, int32_t *s_parent,
                                          int32_t *s_len, int *s_max, bool report) {
  const TablesArgs &t = a.t;
  if (threadIdx.x == 0)
    *s_max = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < a.per; i += blockDim.x) {
    int p = a.parents[base + i];
    const int len = t.lens[base + i];
    if (p != -1 && (p < base || p >= base + a.per)) {
      if (report)
        flag(t.dev_err, GKV_DEVERR_BLOCK_ID);
      p = base + i;
    }
    s_parent[i] = p < 0 ? -1 : p - base;
    s_len[i] = sane(len, t.stride);
    if (s_len[i] != len && report)
      flag(t.dev_err, GKV_DEVERR_LENGTH);
    atomicMax(s_max, blocks_of(s_len[i]));
  }
  __syncthreads();
  return *s_max;
}

// The lengths follow, and the blocks that all rows share are counted: fewer than first, where
// rows are known to differ.
__device__ __forceinline__ void finish_group(const ReorderArgs &a, int group, const int32_t *s_parent,
                                             const int32_t *s_len, int *s_min, int first) {
  const int base = group * a.per;
  if (threadIdx.x == 0)
    *s_min = first;
  __syncthreads();
  for (int i = threadIdx.x; i < a.per; i += blockDim.x) {
    const int len = s_parent[i] < 0 ? 0 : s_len[s_parent[i]];
    a.t.lens[base + i] = len;
    atomicMin(s_min, len / kBlockTokens);
  }
  __syncthreads();
  if (threadIdx.x == 0 && a.shared)
    a.shared[group] = *s_min;
}

// Tiles of columns: the rows' entries go to LDS, and each row takes its parent's from
// there, so it works in place. A row's block gets as many more holders as the row has children,
// less one; where all rows hold the same block that adds up to nothing (or what rows without a
// parent take away), and beams share all but their last blocks: one atomic there, or none.
// A thread's entries are loaded together. A workgroup takes a whole group and finishes it, or,
// where groups are few and long, a tile, and another launch finishes. 64 groups of 16 rows of
// 250 blocks 10.4 us: 4.2 without the table, 4.6 for its entries and 1.8 for the atomics; loads
// of a tile ahead, and ones before the lengths are known, ran level. A group of 16 rows of 6258
// 7.6, and 6 for the second launch.
constexpr int kTileEntries = 1 << 13;
constexpr int kTileParts = kTileEntries / kTableThreads;
__global__ __launch_bounds__(kTableThreads) void tables_reorder_kernel(ReorderArgs a) {
  extern __shared__ int32_t s_mem[];
  const TablesArgs &t = a.t;
  const int width = 1 << a.width_log;
  int32_t *s_tile = s_mem, *s_parent = s_mem + a.per * width, *s_len = s_parent + a.per;
  int32_t *s_more = s_len + a.per; // children of a row, less one
  __shared__ uint8_t s_differ[kTileEntries]; // per column of the tile: not all rows hold the same
  __shared__ int s_max, s_min, s_first, s_sum;
  const int tid = threadIdx.x, group = blockIdx.x / a.tiles, tile = blockIdx.x % a.tiles;
  const int base = group * a.per;
  if (tid == 0) {
    s_first = INT32_MAX;
    s_sum = 0;
  }
  for (int i = tid; i < a.per; i += kTableThreads)
    s_more[i] = -1;
  const int cols = load_group(a, base, s_parent, s_len, &s_max, a.tiles == 1);
  for (int i = tid; i < a.per; i += kTableThreads) {
    if (s_parent[i] >= 0)
      atomicAdd(&s_more[s_parent[i]], 1);
    else
      atomicSub(&s_sum, 1);
  }
  for (int c0 = tile * width; c0 < cols; c0 += a.tiles * width) {
    int32_t was[kTileParts];
#pragma unroll
    for (int k = 0; k < kTileParts; k++) {
      const int e = tid + k * kTableThreads, i = e >> a.width_log, c = c0 + (e & (width - 1));
      was[k] = -1;
      if (i < a.per && c < cols && c < blocks_of(s_len[i]))
        was[k] = t.table[(int64_t)(base + i) * t.stride + c];
    }
    for (int c = tid; c < width; c += kTableThreads)
      s_differ[c] = 0;
#pragma unroll
    for (int k = 0; k < kTileParts; k++) {
      const int e = tid + k * kTableThreads;
      if (e < a.per << a.width_log && c0 + (e & (width - 1)) < cols)
        s_tile[e] = was[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kTileParts; k++) {
      const int e = tid + k * kTableThreads, c = e & (width - 1);
      if (e < a.per << a.width_log && c0 + c < cols && was[k] != s_tile[c])
        s_differ[c] = 1;
    }
    __syncthreads();
    const int p0 = s_parent[0];
#pragma unroll
    for (int k = 0; k < kTileParts; k++) {
      const int e = tid + k * kTableThreads, i = e >> a.width_log, c = e & (width - 1);
      if (i >= a.per || c0 + c >= cols)
        continue;
      const int p = s_parent[i], now = p < 0 ? -1 : s_tile[(p << a.width_log) + c];
      if (now != was[k])
        t.table[(int64_t)(base + i) * t.stride + c0 + c] = now;
      const int more = s_differ[c] ? s_more[i] : i == 0 ? s_sum : 0;
      if (more != 0 && (uint32_t)was[k] < (uint32_t)t.num_blocks)
        atomicAdd(t.refs + was[k], more);
      // (one atomic a wave, whose lanes hold columns in order: thousands on one word of LDS
      // would be served one after another)
      const bool other = now != (p0 < 0 ? -1 : s_tile[(p0 << a.width_log) + c]);
      const uint64_t others = __ballot(other);
      if (other && (width < 64 || (tid & 63) == __ffsll((unsigned long long)others) - 1))
        atomicMin(&s_first, c0 + c);
    }
    __syncthreads();
  }
  if (a.tiles == 1)
    finish_group(a, group, s_parent, s_len, &s_min, s_first);
}

// The second launch where a group has several workgroups: its lengths, and the first column in
// which the new rows differ, up to where the shortest ends.
__global__ __launch_bounds__(kTableThreads) void tables_finish_kernel(ReorderArgs a) {
  extern __shared__ int32_t s_mem[];
  int32_t *s_parent = s_mem, *s_len = s_parent + a.per;
  __shared__ int s_max, s_min, s_first;
  const int base = blockIdx.x * a.per;
  if (threadIdx.x == 0)
    s_first = INT32_MAX;
  load_group(a, base, s_parent, s_len, &s_max, true);
  if (threadIdx.x == 0)
    s_min = INT32_MAX;
  __syncthreads();
  for (int i = threadIdx.x; i < a.per; i += kTableThreads)
    atomicMin(&s_min, s_parent[i] < 0 ? 0 : s_len[s_parent[i]] / kBlockTokens);
  __syncthreads();
  const int full = s_min;
  const int32_t *row = a.t.table + (int64_t)base * a.t.stride;
  // (the columns of a round at once; the first round in which two differ is the last)
  for (int c0 = 0; a.shared && c0 < full; c0 += kTableThreads) {
    const int c = c0 + threadIdx.x;
    if (c < full) {
      const int32_t x = row[c];
      bool same = true;
#pragma unroll 8
      for (int i = 1; i < a.per; i++)
        same &= row[(int64_t)i * a.t.stride + c] == x;
      const uint64_t others = __ballot(!same); // (one atomic a wave)
      if (!same && (int)(threadIdx.x & 63) == __ffsll((unsigned long long)others) - 1)
        atomicMin(&s_first, c);
    }
    __syncthreads();
    const bool found = s_first != INT32_MAX;
    __syncthreads(); // (nobody writes it again before all have looked)
    if (found)
      break;
  }
  __syncthreads();
  finish_group(a, blockIdx.x, s_parent, s_len, &s_min, s_first);
}

// ---- host side ------------------------------------------------------------------------

constexpr int kRowMost = 1 << 17; // blocks of a row: 2 million tokens
constexpr int kReorderWgs = 512; // workgroups that a reorder of few long groups aims at

// What one workgroup carries out by itself: four sequences a wave, four rows a thread.
constexpr int kAloneSeqs = 64, kAloneRows = 4096;

static int tables_check(const gkv_tables &t) {
  if (!t.table || !t.lens || !t.refs || t.table_stride <= 0 || t.n_seqs < 0 || t.num_blocks <= 0)
    return GKV_ERR_ARG;
  if (((uintptr_t)t.table | (uintptr_t)t.lens | (uintptr_t)t.refs) % 4 != 0)
    return GKV_ERR_ARG;
  if (t.table_stride > kRowMost) // (a thousand rows' sums in 32 bits)
    return GKV_ERR_UNSUPPORTED;
  return GKV_OK;
}

static TablesArgs tables_args(const gkv_tables &t, uint32_t *dev_err) {
  return TablesArgs{t.table, t.lens, t.refs, t.table_stride, t.n_seqs, t.num_blocks, dev_err};
}

struct TablesWorkspace {
  size_t old, first, cu, ids, total; // (the flag comes first)
};
static TablesWorkspace tables_workspace(int32_t n_seqs, int32_t num_blocks) {
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  TablesWorkspace w;
  w.old = 256;
  w.first = w.old + up((size_t)n_seqs * 4);
  w.cu = w.first + up((size_t)n_seqs * 4);
  w.ids = w.cu + up(((size_t)n_seqs + 1) * 4);
  w.total = w.ids + (size_t)num_blocks * 4;
  return w;
}

} // namespace gkv

extern "C" int gkv_tables_init(void *stream, gkv_tables t) {
  using namespace gkv;
  const int st = tables_check(t);
  if (st != GKV_OK)
    return st;
  const int64_t n = std::max<int64_t>((int64_t)t.n_seqs * t.table_stride, t.num_blocks);
  const int64_t wgs = std::min<int64_t>((n + 255) / 256, 4096);
  hipLaunchKernelGGL(tables_init_kernel, dim3((unsigned)wgs), dim3(256), 0, (hipStream_t)stream,
                     tables_args(t, nullptr));
  return launch_status("tables_init_kernel");
}

extern "C" size_t gkv_tables_workspace_bytes(int32_t n_seqs, int32_t num_blocks) {
  if (n_seqs < 0 || num_blocks <= 0)
    return 0;
  return gkv::tables_workspace(n_seqs, num_blocks).total;
}

extern "C" int gkv_tables_resize(void *stream, gkv_tables t, const int32_t *new_lens,
                                 int32_t *copy_src, int32_t *copy_dst, int32_t max_rows,
                                 int32_t *cu_rows, int32_t *row_seq, int32_t *row_pos,
                                 int64_t *row_slot, void *workspace, size_t workspace_bytes,
                                 uint32_t *dev_err) {
  using namespace gkv;
  int st = tables_check(t);
  if (st != GKV_OK)
    return st;
  const bool maps = row_seq || row_pos || row_slot;
  if (!new_lens || (copy_src == nullptr) != (copy_dst == nullptr) || max_rows < 0)
    return GKV_ERR_ARG;
  if (((uintptr_t)new_lens | (uintptr_t)copy_src | (uintptr_t)copy_dst | (uintptr_t)cu_rows |
       (uintptr_t)row_seq | (uintptr_t)row_pos) % 4 != 0 || (uintptr_t)row_slot % 8 != 0 ||
      (uintptr_t)workspace % 16 != 0)
    return GKV_ERR_ARG;
  const TablesWorkspace w = tables_workspace(t.n_seqs, t.num_blocks);
  if (!workspace || workspace_bytes < w.total)
    return GKV_ERR_WORKSPACE;
  char *ws = (char *)workspace;
  ResizeArgs a{};
  a.t = tables_args(t, dev_err);
  a.new_lens = new_lens;
  a.copy_src = copy_src;
  a.copy_dst = copy_dst;
  a.max_rows = maps ? max_rows : INT32_MAX;
  a.cu_rows = cu_rows;
  a.row_seq = row_seq;
  a.row_pos = row_pos;
  a.row_slot = row_slot;
  a.maps = maps;
  a.alone = t.n_seqs <= kAloneSeqs && (!maps || max_rows <= kAloneRows);
  a.ok = (int32_t *)ws;
  a.old = (int32_t *)(ws + w.old);
  a.first = (int32_t *)(ws + w.first);
  a.cu = (int32_t *)(ws + w.cu);
  a.ids = (int32_t *)(ws + w.ids);
  const int seq_wgs = (int)(((int64_t)t.n_seqs + 3) / 4);
  const int64_t wgs = seq_wgs + (maps ? ((int64_t)max_rows + 255) / 256 : 0);
  if (!grid_fits(wgs, 256))
    return GKV_ERR_UNSUPPORTED;
  hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(tables_plan_kernel, dim3(1), dim3(kTableThreads), 0, s, a);
  if ((st = launch_status("tables_plan_kernel")) || a.alone)
    return st;
  hipLaunchKernelGGL(tables_apply_kernel, dim3((unsigned)wgs), dim3(256), 0, s, a, seq_wgs);
  return launch_status("tables_apply_kernel");
}

extern "C" int gkv_tables_reorder(void *stream, gkv_tables t, int32_t group_size,
                                  const int32_t *parents, int32_t *shared_blocks,
                                  uint32_t *dev_err) {
  using namespace gkv;
  int st = tables_check(t);
  if (st != GKV_OK)
    return st;
  if (!parents || group_size <= 0 || t.n_seqs % group_size != 0 ||
      ((uintptr_t)parents | (uintptr_t)shared_blocks) % 4 != 0)
    return GKV_ERR_ARG;
  if (group_size > kTileEntries / 4)
    return GKV_ERR_UNSUPPORTED;
  if (t.n_seqs == 0)
    return GKV_OK;
  const int groups = t.n_seqs / group_size;
  ReorderArgs a{};
  a.t = tables_args(t, dev_err);
  a.parents = parents;
  a.per = group_size;
  a.shared = shared_blocks;
  while ((group_size << (a.width_log + 1)) <= kTileEntries && 1 << a.width_log < t.table_stride)
    a.width_log++;
  a.tiles = 1;
  auto tiles = [&]() { return (((int64_t)t.table_stride - 1) >> a.width_log) + 1; };
  if (tiles() > 2 && groups < kReorderWgs) {
    // (narrower tiles where they would be fewer than the CUs: 16 rows of 6258 blocks, 13 of 512
    // columns 17 us, 98 of 64 7.6)
    while (a.width_log > 6 && groups * tiles() < kReorderWgs / 2)
      a.width_log--;
    a.tiles = (int)std::min<int64_t>(tiles(), (kReorderWgs + groups - 1) / groups);
  }
  const int width = 1 << a.width_log;
  const int64_t wgs = (int64_t)groups * a.tiles;
  if (!grid_fits(wgs, kTableThreads))
    return GKV_ERR_UNSUPPORTED;
  const size_t rows = 3 * (size_t)group_size * 4;
  hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(tables_reorder_kernel, dim3((unsigned)wgs), dim3(kTableThreads),
                     (size_t)width * group_size * 4 + rows, s, a);
  if (a.tiles == 1)
    return launch_status("tables_reorder_kernel");
  if ((st = launch_status("tables_reorder_kernel")))
    return st;
  hipLaunchKernelGGL(tables_finish_kernel, dim3((unsigned)groups), dim3(kTableThreads), rows, s, a);
  return launch_status("tables_finish_kernel");
}
