// Paged KV pool: device storage of every layer's cache plus the host
// bookkeeping of blocks and sequences.
//
// Replaces the reference engine's per-layer contiguous caches
// (GpuLayer::kc16/vq8/vs, getp-csrc/engine/gpu_engine.hpp:59-78, allocated in
// gpu_alloc_state :316-334 with slots = max_pos or the window, rounded to 64)
// by 16-token blocks handed out from a free list:
//   full layers    one block id covers 16 positions of a sequence in every full
//                  layer; per layer K and V [num_blocks][Hkv][1024] bf16 in
//                  the block layouts of kv_append.hpp (32 KB per block at Hkv=8)
//   window layers  a ring of W/16 blocks per sequence id, fixed at create time
//                  (the reference's slots = window, gpu_engine.hpp:318-319); a
//                  pool that keeps first tokens: kept/16 + W/16 + 1 blocks
//   sharing        a fork holds its parent's full blocks too: every block counts
//                  its holders and returns to the free list with the last one;
//                  the partly filled last block is copied, so that nobody
//                  appends to a block that another sequence reads
//   tables         int32 [max_seqs][ceil(max_seq_len/16)] and [max_seqs][W/16],
//                  mirrored on the host; gkv_pool_sync uploads the entries that
//                  changed since the last sync, without waiting
// Sizing: num_blocks explicit, or derived from a byte budget, by default 90%
// of the free device memory (288 GB HBM3E on MI355X), instead of the
// reference's halve-the-batch-until-it-fits loop (gpu_fit_batch :425-433).
// Errors are returned, never exit()ed (the reference's HIP_CHECK exits,
// :41-49).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <cstring>
#include <exception>
#include <memory>
#include <numeric>
#include <random>
#include <vector>

#include "block_copy.hpp"
#include "gkv.h"

namespace {
constexpr int kBT = 16;
constexpr int kD = 64;
} // namespace

struct gkv_pool {
  gkv_pool_config cfg{};
  std::vector<int> layer_index; // layer -> index among full or window layers
  std::vector<char> layer_is_window;
  int n_full = 0, n_window = 0;
  int table_stride = 0; // full-table entries per sequence
  int ring_blocks = 0;  // window layers' table entries per sequence: W / 16, or kept / 16 + W / 16 + 1
  int ring = 0;         // slots of the window layers' ring: W, or W + 16
  int kept = 0;         // positions before it that stay
  int64_t num_blocks = 0, num_ring_blocks = 0;
  std::vector<void *> k_full, v_full, k_ring, v_ring;
  std::vector<void *> s_full, s_ring; // fp32 V scales (int8 V only)
  int32_t *d_table = nullptr, *d_ring_table = nullptr;
  std::vector<int32_t> h_table, h_ring_table;
  std::vector<int32_t> free_blocks; // stack; back() is handed out next
  std::vector<int32_t> refs;        // per block: the sequences that hold it
  std::vector<int32_t> seq_blocks;  // blocks held per sequence
  // What the window layers' rings hold, for forks and trims that go back: units of
  // `unit` tokens (16; 1 in a ring of W slots, where a token takes another's place alone),
  // per sequence the unit in each place when it was forked or last trimmed, its length then,
  // and its length now by the last reserve.
  int unit = 1, units = 0;
  std::vector<int32_t> ring_units, seq_base, seq_len;
  std::vector<char> seq_live;
  std::vector<int32_t> free_seqs;
  int64_t device_bytes = 0;
  // Incremental sync: the full-table entries changed since the last sync,
  // as (index, value); they go to the device through one of two pinned
  // staging buffers (reused only once the copy out of it has completed) and
  // a scatter kernel. The first sync uploads the whole tables.
  std::vector<int2> pending;
  bool whole = true;
  int2 *h_stage[2] = {nullptr, nullptr};
  int2 *d_stage[2] = {nullptr, nullptr};
  hipEvent_t stage_done[2] = {nullptr, nullptr};
  size_t stage_cap = 0; // entries per staging buffer
  int stage_i = 0;

  void free_stage() {
    for (int i = 0; i < 2; i++) {
      if (stage_done[i]) {
        (void)hipEventSynchronize(stage_done[i]);
        (void)hipEventDestroy(stage_done[i]);
      }
      if (h_stage[i])
        (void)hipHostFree(h_stage[i]);
      if (d_stage[i])
        (void)hipFree(d_stage[i]);
      h_stage[i] = nullptr;
      d_stage[i] = nullptr;
      stage_done[i] = nullptr;
    }
    stage_cap = 0;
  }

  // Room for n more changed entries, made before a call takes anything.
  void make_room(size_t n) {
    if (pending.size() + n > pending.capacity())
      pending.reserve(std::max(pending.size() + n, 2 * pending.capacity()));
  }

  // The staging buffer for the next n pairs (grown if need be), free to be
  // filled: its previous copy (two uses ago) has long completed in practice,
  // the wait only guards the case where it has not.
  int stage_for(size_t n, int *k) {
    if (n > stage_cap) {
      free_stage();
      const size_t cap = std::max<size_t>(n, 4096);
      for (int i = 0; i < 2; i++)
        if (hipHostMalloc((void **)&h_stage[i], cap * sizeof(int2), hipHostMallocDefault) !=
                hipSuccess ||
            hipMalloc((void **)&d_stage[i], cap * sizeof(int2)) != hipSuccess ||
            hipEventCreateWithFlags(&stage_done[i], hipEventDisableTiming) != hipSuccess) {
          free_stage();
          return GKV_ERR_HIP;
        }
      stage_cap = cap;
    }
    *k = stage_i;
    return hipEventSynchronize(stage_done[stage_i]) == hipSuccess ? GKV_OK : GKV_ERR_HIP;
  }

  gkv_cache_view layer_view(int layer) const {
    const int i = layer_index[layer];
    gkv_cache_view v{};
    v.n_kv_heads = cfg.n_kv_heads;
    v.v_format = cfg.v_format;
    if (layer_is_window[layer]) {
      v.k = k_ring[i];
      v.v = v_ring[i];
      v.v_scale = s_ring[i];
      v.block_table = d_ring_table;
      v.table_stride = ring_blocks;
      v.num_blocks = (int32_t)num_ring_blocks;
      v.ring = ring;
    } else {
      v.k = k_full[i];
      v.v = v_full[i];
      v.v_scale = s_full[i];
      v.block_table = d_table;
      v.table_stride = table_stride;
      v.num_blocks = (int32_t)num_blocks;
    }
    return v;
  }

  // The unit that place e of a sequence's ring holds when the sequence is len tokens long:
  // the last one appended there since its base, or what was there then.
  int32_t ring_unit(int32_t seq, int32_t e, int32_t len) const {
    const int32_t kept_units = kept / unit, last = (len - 1) / unit, back = last - kept_units - e;
    if (len > seq_base[seq] && back >= 0) {
      const int32_t u = last - back % units;
      if (u >= seq_base[seq] / unit)
        return u;
    }
    return ring_units[(size_t)seq * units + e];
  }

  // Whether the rings of a sequence of len tokens hold what the token behind its
  // first n sees of them: positions max(n - W + 1, kept) .. n - 1.
  bool ring_holds(int32_t seq, int32_t n, int32_t len) const {
    const int32_t first = std::max({n - cfg.window + 1, kept, 0});
    if (n_window == 0 || first >= n)
      return true;
    for (int32_t u = first / unit; u <= (n - 1) / unit; u++)
      if (ring_unit(seq, (u - kept / unit) % units, len) != u)
        return false;
    return true;
  }

  // Sequence `to` goes on at n tokens, with the rings of `from` (a sequence of len).
  void ring_rebase(int32_t to, int32_t from, int32_t n, int32_t len) {
    if (to == from && n >= seq_len[to])
      return; // (nothing dropped)
    if (n_window > 0)
      for (int32_t e = 0; e < units; e++)
        ring_units[(size_t)to * units + e] = ring_unit(from, e, len);
    seq_base[to] = seq_len[to] = n;
  }

  // Copies blocks {src, dst} in every full (or window) layer, on stream: one
  // launch per 32 layers. The ids travel as kernel arguments, or, many of
  // them, through a staging buffer.
  int copy(const std::vector<int2> &pairs, bool window, hipStream_t s) {
    std::vector<gkv_cache_view> views;
    for (int l = 0; l < cfg.n_layers; l++)
      if ((layer_is_window[l] != 0) == window)
        views.push_back(layer_view(l));
    const int n = (int)pairs.size(), n_views = (int)views.size();
    if (n == 0 || n_views == 0)
      return GKV_OK;
    if (n <= gkv::kInlinePairs)
      return gkv::copy_blocks(s, views.data(), n_views, n, nullptr, nullptr, 0, pairs.data(),
                              nullptr);
    int k = 0;
    int st = stage_for(pairs.size(), &k);
    if (st != GKV_OK)
      return st;
    std::memcpy(h_stage[k], pairs.data(), pairs.size() * sizeof(int2));
    if (hipMemcpyAsync(d_stage[k], h_stage[k], pairs.size() * sizeof(int2), hipMemcpyHostToDevice,
                       s) != hipSuccess)
      return GKV_ERR_HIP;
    st = gkv::copy_blocks(s, views.data(), n_views, n, (const int32_t *)d_stage[k],
                          (const int32_t *)d_stage[k] + 1, 2, nullptr, nullptr);
    if (hipEventRecord(stage_done[k], s) != hipSuccess)
      st = GKV_ERR_HIP;
    stage_i ^= 1;
    return st;
  }

  ~gkv_pool() {
    free_stage();
    for (auto *vec : {&k_full, &v_full, &k_ring, &v_ring, &s_full, &s_ring})
      for (void *p : *vec)
        if (p)
          (void)hipFree(p);
    if (d_table)
      (void)hipFree(d_table);
    if (d_ring_table)
      (void)hipFree(d_ring_table);
  }
};

static int pool_create(const gkv_pool_config *cfg, int32_t kept, int32_t slack, gkv_pool **out) try {
  if (!cfg || !out)
    return GKV_ERR_ARG;
  *out = nullptr;
  const gkv_pool_config &c = *cfg;
  if (c.n_layers <= 0 || c.n_kv_heads <= 0 || c.max_seqs <= 0 || c.max_seq_len <= 0 ||
      c.window < 0 || c.num_blocks < 0 || c.bytes_budget < 0)
    return GKV_ERR_ARG;
  if (c.head_dim != kD || c.window % kBT != 0)
    return GKV_ERR_UNSUPPORTED;
  gkv::BlockBytes bb;
  if (c.n_kv_heads > 65536 || gkv::block_bytes(c.n_kv_heads, c.v_format, &bb) != GKV_OK)
    return GKV_ERR_ARG;
  std::unique_ptr<gkv_pool> p(new gkv_pool());
  p->cfg = c;
  p->layer_index.resize(c.n_layers);
  p->layer_is_window.resize(c.n_layers);
  for (int l = 0; l < c.n_layers; l++) {
    const bool win = c.window > 0 && l % 2 == 0; // run.cpp:617 (l % 2 == 0)
    p->layer_is_window[l] = win;
    p->layer_index[l] = win ? p->n_window++ : p->n_full++;
  }
  p->table_stride = (c.max_seq_len + kBT - 1) / kBT;
  p->ring = c.window > 0 ? c.window + slack : 0;
  p->kept = kept;
  p->ring_blocks = c.window > 0 ? (kept + c.window + slack) / kBT : 0;
  p->num_ring_blocks = (int64_t)c.max_seqs * p->ring_blocks;
  const int64_t bpl = bb.k + bb.v + bb.s;
  const int64_t ring_bytes = p->num_ring_blocks * bpl * p->n_window;
  const int64_t table_bytes =
      ((int64_t)c.max_seqs * p->table_stride + (int64_t)c.max_seqs * p->ring_blocks) * 4;

  int64_t nb = c.num_blocks;
  if (nb == 0 && p->n_full > 0) {
    int64_t budget = c.bytes_budget;
    if (budget == 0) {
      size_t free_b = 0, total_b = 0;
      if (hipMemGetInfo(&free_b, &total_b) != hipSuccess)
        return GKV_ERR_HIP;
      budget = (int64_t)(0.9 * (double)free_b);
    }
    nb = (budget - ring_bytes - table_bytes) / (bpl * p->n_full);
    if (nb <= 0)
      return GKV_ERR_CAPACITY;
  }
  if (nb > INT32_MAX || p->num_ring_blocks > INT32_MAX)
    return GKV_ERR_CAPACITY;
  p->num_blocks = p->n_full > 0 ? nb : 0;

  auto dev_alloc = [&](void **ptr, int64_t bytes) -> bool {
    if (bytes == 0) {
      *ptr = nullptr;
      return true;
    }
    if (hipMalloc(ptr, (size_t)bytes) != hipSuccess) {
      *ptr = nullptr;
      (void)hipGetLastError();
      return false;
    }
    p->device_bytes += bytes;
    return true;
  };
  const int64_t kb = bb.k, vb = bb.v, sb = bb.s;
  bool ok = true;
  p->k_full.assign(p->n_full, nullptr);
  p->v_full.assign(p->n_full, nullptr);
  p->s_full.assign(p->n_full, nullptr);
  p->k_ring.assign(p->n_window, nullptr);
  p->v_ring.assign(p->n_window, nullptr);
  p->s_ring.assign(p->n_window, nullptr);
  for (int i = 0; ok && i < p->n_full; i++)
    ok = dev_alloc(&p->k_full[i], p->num_blocks * kb) &&
         dev_alloc(&p->v_full[i], p->num_blocks * vb) &&
         dev_alloc(&p->s_full[i], p->num_blocks * sb);
  for (int i = 0; ok && i < p->n_window; i++)
    ok = dev_alloc(&p->k_ring[i], p->num_ring_blocks * kb) &&
         dev_alloc(&p->v_ring[i], p->num_ring_blocks * vb) &&
         dev_alloc(&p->s_ring[i], p->num_ring_blocks * sb);
  ok = ok && dev_alloc((void **)&p->d_table, (int64_t)c.max_seqs * p->table_stride * 4);
  if (ok && p->ring_blocks > 0)
    ok = dev_alloc((void **)&p->d_ring_table, (int64_t)c.max_seqs * p->ring_blocks * 4);
  if (!ok)
    return GKV_ERR_CAPACITY;

  // Unassigned table entries are -1: a kernel that meets one flags it.
  p->h_table.assign((size_t)c.max_seqs * p->table_stride, -1);
  p->h_ring_table.resize((size_t)c.max_seqs * p->ring_blocks);
  std::vector<int32_t> ring_ids(p->num_ring_blocks);
  std::iota(ring_ids.begin(), ring_ids.end(), 0);
  p->free_blocks.resize(p->num_blocks);
  // Stack order: block 0 is handed out first unless shuffled.
  for (int64_t i = 0; i < p->num_blocks; i++)
    p->free_blocks[i] = (int32_t)(p->num_blocks - 1 - i);
  if (c.shuffle_seed != 0) {
    std::mt19937_64 rng(c.shuffle_seed);
    std::shuffle(p->free_blocks.begin(), p->free_blocks.end(), rng);
    std::shuffle(ring_ids.begin(), ring_ids.end(), rng);
  }
  std::copy(ring_ids.begin(), ring_ids.end(), p->h_ring_table.begin());
  p->refs.assign(p->num_blocks, 0);
  p->seq_blocks.assign(c.max_seqs, 0);
  p->unit = slack > 0 ? kBT : 1;
  p->units = p->ring / p->unit;
  p->ring_units.assign((size_t)c.max_seqs * p->units, -1);
  p->seq_base.assign(c.max_seqs, 0);
  p->seq_len.assign(c.max_seqs, 0);
  p->seq_live.assign(c.max_seqs, 0);
  p->free_seqs.resize(c.max_seqs);
  for (int s = 0; s < c.max_seqs; s++)
    p->free_seqs[s] = c.max_seqs - 1 - s;
  if (gkv_pool_sync(p.get(), nullptr) != GKV_OK || hipDeviceSynchronize() != hipSuccess)
    return GKV_ERR_HIP;
  *out = p.release();
  return GKV_OK;
} catch (const std::exception &) {
  return GKV_ERR_CAPACITY; // out of host memory
}

extern "C" int gkv_pool_create(const gkv_pool_config *cfg, gkv_pool **out) {
  // the block format's scale needs whole blocks to leave a window at once
  if (cfg && cfg->v_format == GKV_KV_FP8_BLOCK && cfg->window > 0) {
    if (out)
      *out = nullptr;
    return GKV_ERR_UNSUPPORTED;
  }
  return pool_create(cfg, 0, 0, out);
}

extern "C" int gkv_pool_create_kept(const gkv_pool_config *cfg, int32_t kept, gkv_pool **out) {
  if (!cfg || !out)
    return GKV_ERR_ARG;
  *out = nullptr;
  if (kept < 0 || kept > INT32_MAX / 4 || cfg->window <= 0 || cfg->window > INT32_MAX / 4)
    return GKV_ERR_ARG;
  if (kept % kBT != 0)
    return GKV_ERR_UNSUPPORTED;
  if (cfg->v_format != GKV_V_BF16 && cfg->v_format != GKV_KV_FP8_BLOCK)
    return GKV_ERR_UNSUPPORTED; // what the gkv_kept_* entry points read
  return pool_create(cfg, kept, kBT, out);
}

extern "C" int gkv_pool_destroy(gkv_pool *pool) {
  if (!pool)
    return GKV_ERR_ARG;
  (void)hipDeviceSynchronize();
  delete pool;
  return GKV_OK;
}

extern "C" int gkv_pool_seq_alloc(gkv_pool *pool, int32_t *seq_id) {
  if (!pool || !seq_id)
    return GKV_ERR_ARG;
  if (pool->free_seqs.empty())
    return GKV_ERR_CAPACITY;
  const int32_t s = pool->free_seqs.back();
  pool->free_seqs.pop_back();
  pool->seq_live[s] = 1;
  pool->seq_blocks[s] = 0;
  pool->seq_base[s] = pool->seq_len[s] = 0;
  std::fill_n(pool->ring_units.begin() + (size_t)s * pool->units, pool->units, -1);
  *seq_id = s;
  return GKV_OK;
}

extern "C" int gkv_pool_seq_reserve(gkv_pool *pool, int32_t seq_id, int32_t seq_len) try {
  if (!pool || seq_len < 0)
    return GKV_ERR_ARG;
  if (seq_id < 0 || seq_id >= pool->cfg.max_seqs || !pool->seq_live[seq_id])
    return GKV_ERR_BLOCK;
  const int32_t len = std::max(seq_len, pool->seq_base[seq_id]);
  if (pool->n_full == 0) {
    if (seq_len > pool->cfg.max_seq_len)
      return GKV_ERR_CAPACITY;
    pool->seq_len[seq_id] = len;
    return GKV_OK;
  }
  const int32_t need = (seq_len + kBT - 1) / kBT;
  if (need > pool->table_stride)
    return GKV_ERR_CAPACITY;
  const int32_t have = pool->seq_blocks[seq_id];
  if (need <= have) {
    pool->seq_len[seq_id] = len;
    return GKV_OK;
  }
  if ((int64_t)(need - have) > (int64_t)pool->free_blocks.size())
    return GKV_ERR_CAPACITY; // nothing taken: all or none
  pool->make_room(need - have);
  const size_t base = (size_t)seq_id * pool->table_stride;
  int32_t *row = &pool->h_table[base];
  for (int32_t j = have; j < need; j++) {
    row[j] = pool->free_blocks.back();
    pool->free_blocks.pop_back();
    pool->refs[row[j]] = 1;
    pool->pending.push_back(int2{(int)(base + j), row[j]});
  }
  pool->seq_blocks[seq_id] = need;
  pool->seq_len[seq_id] = len;
  return GKV_OK;
} catch (const std::exception &) {
  return GKV_ERR_CAPACITY; // out of host memory
}

extern "C" int gkv_pool_seq_free(gkv_pool *pool, int32_t seq_id) try {
  if (!pool)
    return GKV_ERR_ARG;
  if (seq_id < 0 || seq_id >= pool->cfg.max_seqs || !pool->seq_live[seq_id])
    return GKV_ERR_BLOCK;
  const size_t base = (size_t)seq_id * pool->table_stride;
  int32_t *row = &pool->h_table[base];
  pool->make_room(pool->seq_blocks[seq_id]);
  for (int32_t j = pool->seq_blocks[seq_id] - 1; j >= 0; j--) {
    if (--pool->refs[row[j]] == 0) // (the capacity for every block is there)
      pool->free_blocks.push_back(row[j]);
    row[j] = -1;
    pool->pending.push_back(int2{(int)(base + j), -1});
  }
  pool->seq_blocks[seq_id] = 0;
  pool->seq_live[seq_id] = 0;
  pool->free_seqs.push_back(seq_id);
  return GKV_OK;
} catch (const std::exception &) {
  return GKV_ERR_CAPACITY; // out of host memory
}

// ---- sharing, trimming, compacting ---------------------------------------------
//
// The copies go out on the caller's stream at once, the table entries with the
// next gkv_pool_sync on it. Nothing is taken before the copies are queued, so
// a failed call leaves the bookkeeping as it was.

extern "C" int gkv_pool_seq_fork(gkv_pool *pool, int32_t parent, int32_t n_tokens, void *stream,
                                 int32_t *child) try {
  if (!pool || !child || n_tokens < 0)
    return GKV_ERR_ARG;
  if (parent < 0 || parent >= pool->cfg.max_seqs || !pool->seq_live[parent])
    return GKV_ERR_BLOCK;
  const int32_t shared = n_tokens / kBT, part = n_tokens % kBT != 0;
  if (n_tokens > pool->cfg.max_seq_len ||
      (pool->n_full > 0 && shared + part > pool->seq_blocks[parent]))
    return GKV_ERR_ARG; // more tokens than the parent holds
  const int32_t len = std::max(pool->seq_len[parent], n_tokens);
  if (!pool->ring_holds(parent, n_tokens, len))
    return GKV_ERR_ARG; // the child's next token would see what the parent's later ones replaced
  const bool full = pool->n_full > 0;
  if (pool->free_seqs.empty() || (full && part && pool->free_blocks.empty()))
    return GKV_ERR_CAPACITY;
  const int32_t id = pool->free_seqs.back();
  const size_t from = (size_t)parent * pool->table_stride, to = (size_t)id * pool->table_stride;
  if (full)
    pool->make_room(shared + part);
  hipStream_t s = (hipStream_t)stream;
  if (full && part) {
    const int st = pool->copy({int2{pool->h_table[from + shared], pool->free_blocks.back()}}, false, s);
    if (st != GKV_OK)
      return st;
  }
  if (pool->n_window > 0) {
    // the ring's blocks in use (the kept tokens' first), slot by slot
    std::vector<int2> ring;
    const size_t rb = pool->ring_blocks;
    for (size_t j = 0; j < std::min<size_t>(rb, shared + part); j++)
      ring.push_back(int2{pool->h_ring_table[parent * rb + j], pool->h_ring_table[id * rb + j]});
    const int st = pool->copy(ring, true, s);
    if (st != GKV_OK)
      return st;
  }
  if (full) {
    for (int32_t j = 0; j < shared; j++) {
      pool->h_table[to + j] = pool->h_table[from + j];
      pool->refs[pool->h_table[from + j]]++;
    }
    if (part) {
      const int32_t blk = pool->free_blocks.back();
      pool->free_blocks.pop_back();
      pool->refs[blk] = 1;
      pool->h_table[to + shared] = blk;
    }
    for (int32_t j = 0; j < shared + part; j++)
      pool->pending.push_back(int2{(int)(to + j), pool->h_table[to + j]});
    pool->seq_blocks[id] = shared + part;
  } else {
    pool->seq_blocks[id] = 0;
  }
  pool->free_seqs.pop_back();
  pool->seq_live[id] = 1;
  pool->ring_rebase(id, parent, n_tokens, len);
  *child = id;
  return GKV_OK;
} catch (const std::exception &) {
  return GKV_ERR_CAPACITY; // out of host memory
}

extern "C" int gkv_pool_seq_trim(gkv_pool *pool, int32_t seq_id, int32_t n_tokens,
                                 void *stream) try {
  if (!pool || n_tokens < 0)
    return GKV_ERR_ARG;
  if (seq_id < 0 || seq_id >= pool->cfg.max_seqs || !pool->seq_live[seq_id])
    return GKV_ERR_BLOCK;
  const int32_t len = std::max(pool->seq_len[seq_id], n_tokens);
  if (!pool->ring_holds(seq_id, n_tokens, len))
    return GKV_ERR_ARG; // the next token would see what the dropped ones replaced
  if (pool->n_full == 0) {
    pool->ring_rebase(seq_id, seq_id, n_tokens, len);
    return GKV_OK;
  }
  const int32_t have = pool->seq_blocks[seq_id], keep = n_tokens / kBT + (n_tokens % kBT != 0);
  if (keep > have)
    return GKV_ERR_ARG;
  const size_t base = (size_t)seq_id * pool->table_stride;
  int32_t *row = &pool->h_table[base];
  pool->make_room((have - keep) + 1);
  // appends go on inside the last block: it has to be this sequence's own
  int32_t own = -1;
  if (n_tokens % kBT != 0 && pool->refs[row[keep - 1]] > 1) {
    if (!pool->free_blocks.empty())
      own = pool->free_blocks.back();
    for (int32_t j = keep; own < 0 && j < have; j++)
      if (pool->refs[row[j]] == 1)
        own = row[j]; // one of those that this call frees
    if (own < 0)
      return GKV_ERR_CAPACITY;
    const int st = pool->copy({int2{row[keep - 1], own}}, false, (hipStream_t)stream);
    if (st != GKV_OK)
      return st;
  }
  for (int32_t j = have - 1; j >= keep; j--) {
    if (--pool->refs[row[j]] == 0)
      pool->free_blocks.push_back(row[j]);
    row[j] = -1;
    pool->pending.push_back(int2{(int)(base + j), -1});
  }
  if (own >= 0) {
    pool->free_blocks.erase(std::find(pool->free_blocks.begin(), pool->free_blocks.end(), own));
    pool->refs[row[keep - 1]]--;
    pool->refs[own] = 1;
    row[keep - 1] = own;
    pool->pending.push_back(int2{(int)(base + keep - 1), own});
  }
  pool->seq_blocks[seq_id] = keep;
  pool->ring_rebase(seq_id, seq_id, n_tokens, len);
  return GKV_OK;
} catch (const std::exception &) {
  return GKV_ERR_CAPACITY; // out of host memory
}

extern "C" int gkv_pool_compact(gkv_pool *pool, void *stream, int64_t *n_used) try {
  if (!pool)
    return GKV_ERR_ARG;
  const int64_t nb = pool->num_blocks, live = nb - (int64_t)pool->free_blocks.size();
  // block `live` and those behind move into the holes before it: the sources
  // and the targets are disjoint, so the copies need no order
  std::vector<int2> moves;
  std::vector<int32_t> now(nb);
  std::iota(now.begin(), now.end(), 0);
  int32_t hole = 0;
  for (int64_t i = live; i < nb; i++) {
    if (pool->refs[i] == 0)
      continue;
    while (pool->refs[hole] != 0)
      hole++;
    moves.push_back(int2{(int)i, hole});
    now[i] = hole++;
  }
  size_t entries = 0;
  for (int32_t q = 0; q < pool->cfg.max_seqs; q++)
    entries += pool->seq_blocks[q];
  pool->make_room(moves.empty() ? 0 : entries);
  const int st = pool->copy(moves, false, (hipStream_t)stream);
  if (st != GKV_OK)
    return st;
  for (const int2 &m : moves)
    std::swap(pool->refs[m.x], pool->refs[m.y]);
  for (int32_t q = 0; q < pool->cfg.max_seqs; q++) {
    const size_t base = (size_t)q * pool->table_stride;
    for (int32_t j = 0; j < pool->seq_blocks[q]; j++) {
      int32_t &id = pool->h_table[base + j];
      if (now[id] != id) {
        id = now[id];
        pool->pending.push_back(int2{(int)(base + j), id});
      }
    }
  }
  for (int64_t i = 0; i < nb - live; i++) // the lowest free block is handed out next
    pool->free_blocks[i] = (int32_t)(nb - 1 - i);
  if (n_used)
    *n_used = live;
  return GKV_OK;
} catch (const std::exception &) {
  return GKV_ERR_CAPACITY; // out of host memory
}

// Applies n staged (index, value) pairs to the device table, in order (a
// later pair for the same entry wins: each thread takes a distinct pair, and
// the pairs of one entry never repeat within a sync, see gkv_pool_sync).
__global__ void pool_scatter_kernel(int32_t *table, const int2 *pairs, int n) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n)
    table[pairs[i].x] = pairs[i].y;
}

extern "C" int gkv_pool_sync(gkv_pool *pool, void *stream) {
  if (!pool)
    return GKV_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  if (pool->whole) {
    // the first sync: both tables whole, waited for (create time)
    if (hipMemcpyAsync(pool->d_table, pool->h_table.data(), pool->h_table.size() * 4,
                       hipMemcpyHostToDevice, s) != hipSuccess)
      return GKV_ERR_HIP;
    if (pool->d_ring_table &&
        hipMemcpyAsync(pool->d_ring_table, pool->h_ring_table.data(),
                       pool->h_ring_table.size() * 4, hipMemcpyHostToDevice, s) != hipSuccess)
      return GKV_ERR_HIP;
    if (hipStreamSynchronize(s) != hipSuccess)
      return GKV_ERR_HIP;
    pool->whole = false;
    pool->pending.clear();
    return GKV_OK;
  }
  if (pool->pending.empty())
    return GKV_OK;
  // One pair per changed entry, its latest value (a reserve after a free of
  // the same entry within one sync leaves two pairs; the host table holds
  // the value that counts).
  std::vector<int2> &pend = pool->pending;
  std::sort(pend.begin(), pend.end(), [](const int2 &x, const int2 &y) { return x.x < y.x; });
  pend.erase(std::unique(pend.begin(), pend.end(),
                         [](const int2 &x, const int2 &y) { return x.x == y.x; }),
             pend.end());
  for (int2 &e : pend)
    e.y = pool->h_table[e.x];
  const size_t n = pend.size();
  int k = 0;
  const int st = pool->stage_for(n, &k);
  if (st != GKV_OK)
    return st;
  std::memcpy(pool->h_stage[k], pend.data(), n * sizeof(int2));
  if (hipMemcpyAsync(pool->d_stage[k], pool->h_stage[k], n * sizeof(int2), hipMemcpyHostToDevice,
                     s) != hipSuccess)
    return GKV_ERR_HIP;
  hipLaunchKernelGGL(pool_scatter_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s,
                     pool->d_table, pool->d_stage[k], (int)n);
  if (hipGetLastError() != hipSuccess || hipEventRecord(pool->stage_done[k], s) != hipSuccess)
    return GKV_ERR_HIP;
  pool->stage_i ^= 1;
  pend.clear();
  return GKV_OK;
}

extern "C" int gkv_pool_layer_view_from(const gkv_pool *pool, int32_t layer, int32_t first_seq,
                                        gkv_cache_view *view) {
  if (!pool || !view || layer < 0 || layer >= pool->cfg.n_layers || first_seq < 0 ||
      first_seq >= pool->cfg.max_seqs)
    return GKV_ERR_ARG;
  gkv_cache_view v = pool->layer_view(layer);
  v.block_table += (size_t)first_seq * v.table_stride;
  *view = v;
  return GKV_OK;
}

extern "C" int gkv_pool_layer_view(const gkv_pool *pool, int32_t layer, gkv_cache_view *view) {
  return gkv_pool_layer_view_from(pool, layer, 0, view);
}

extern "C" int64_t gkv_pool_free_blocks(const gkv_pool *pool) {
  return pool ? (int64_t)pool->free_blocks.size() : -1;
}

extern "C" int64_t gkv_pool_num_blocks(const gkv_pool *pool) {
  return pool ? pool->num_blocks : -1;
}

extern "C" int64_t gkv_pool_device_bytes(const gkv_pool *pool) {
  return pool ? pool->device_bytes : -1;
}

extern "C" int gkv_pool_seq_blocks(const gkv_pool *pool, int32_t seq_id, int32_t *blocks,
                                   int32_t n, int32_t *n_used) {
  if (!pool || n < 0 || (n > 0 && !blocks))
    return GKV_ERR_ARG;
  if (seq_id < 0 || seq_id >= pool->cfg.max_seqs || !pool->seq_live[seq_id])
    return GKV_ERR_BLOCK;
  const int32_t used = pool->seq_blocks[seq_id];
  const int32_t *row = &pool->h_table[(size_t)seq_id * pool->table_stride];
  for (int32_t j = 0; j < std::min(n, used); j++)
    blocks[j] = row[j];
  if (n_used)
    *n_used = used;
  return GKV_OK;
}
