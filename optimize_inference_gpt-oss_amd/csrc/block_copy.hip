// Copies of whole cache blocks inside a paged cache, in several layers at once:
// the last, partly filled block of a forked sequence, a ring copied to a
// fork's, the blocks that a compaction moves.
//
// A block of one layer is up to three contiguous pieces: K and V (1 or 2 KB a
// head) and the scales. One workgroup copies one (layer, pair), its three pieces
// one behind the other, 16 bytes a thread and load; few pairs are cut
// into parts, so that the copy of a handful of blocks still spreads over the
// CUs. Bound by HBM, each byte read once and written once: 2048 blocks of 12 layers
// (bf16, 8 heads, 1.6 GB read and written) 310 us, 5.2 TB/s, a large copy's rate; 8
// blocks of 12 layers 3.3 us.
#include "block_copy.hpp"

#include <algorithm>
#include <type_traits>

namespace gkv {

constexpr int kCopyThreads = 256;
constexpr int kCopyViews = 32;  // layers per launch (their pointers are kernel arguments)
constexpr int kCopySpread = 1024; // workgroups up to which pairs are cut into parts
constexpr int kCopyParts = 4;
constexpr int kCopyGrid = 1 << 23; // workgroups per launch, at most (a launch takes 2^32 threads)

struct CopyLayer {
  char *k, *v, *s;
  uint32_t k_bytes, v_bytes, s_bytes; // per block; K and V multiples of 16, the scales of 8
  int32_t num_blocks;
};

struct CopyArgs {
  CopyLayer layer[kCopyViews];
  int n_layers, n_pairs, parts;
  const int32_t *src, *dst; // block ids, `stride` apart
  int stride;
  uint32_t *dev_err;
};

struct InlinePairs {
  int2 p[kInlinePairs];
};
struct NoPairs {}; // (a kilobyte of arguments less to hand over)

// n bytes (a multiple of 16) by the threads of one part, four loads in
// flight a thread.
__device__ __forceinline__ void copy_piece(char *dst, const char *src, uint32_t n, int first,
                                           int step) {
  const uint32_t n16 = n / 16;
  for (uint32_t i = first; i < n16; i += 4 * step) {
    u32x4 x[4];
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (i + j * step < n16)
        x[j] = __builtin_nontemporal_load((const u32x4 *)src + i + j * step);
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (i + j * step < n16)
        __builtin_nontemporal_store(x[j], (u32x4 *)dst + i + j * step);
  }
}

template <typename Pairs>
__global__ __launch_bounds__(kCopyThreads) void copy_blocks_kernel(CopyArgs a, Pairs in) {
  // pair fastest, so that the workgroups at work at a time stay in one layer
  const int part = blockIdx.x % a.parts, item = blockIdx.x / a.parts;
  const int pair = item % a.n_pairs;
  const CopyLayer &l = a.layer[item / a.n_pairs];
  int s, d;
  if constexpr (std::is_same_v<Pairs, InlinePairs>) {
    s = in.p[pair].x;
    d = in.p[pair].y;
  } else {
    s = a.src[(int64_t)pair * a.stride];
    d = a.dst[(int64_t)pair * a.stride];
  }
  if (s < 0 || d < 0 || s >= l.num_blocks || d >= l.num_blocks) {
    if (threadIdx.x == 0 && a.dev_err)
      atomicOr(a.dev_err, GKV_DEVERR_BLOCK_ID);
    return;
  }
  if (s == d)
    return;
  const int first = part * kCopyThreads + threadIdx.x, step = a.parts * kCopyThreads;
  copy_piece(l.k + (size_t)d * l.k_bytes, l.k + (size_t)s * l.k_bytes, l.k_bytes, first, step);
  copy_piece(l.v + (size_t)d * l.v_bytes, l.v + (size_t)s * l.v_bytes, l.v_bytes, first, step);
  for (uint32_t i = first; i < l.s_bytes / 8; i += step)
    ((u32x2 *)(l.s + (size_t)d * l.s_bytes))[i] = ((const u32x2 *)(l.s + (size_t)s * l.s_bytes))[i];
}

int block_bytes(int n_kv_heads, int v_format, BlockBytes *out) {
  const int64_t h = n_kv_heads, half = h * kBlockTokens * kHeadDim;
  switch (v_format) {
  case GKV_V_BF16:
    *out = BlockBytes{2 * half, 2 * half, 0};
    return GKV_OK;
  case GKV_V_INT8:
    *out = BlockBytes{2 * half, half, h * kBlockTokens * 4};
    return GKV_OK;
  case GKV_KV_FP8:
    *out = BlockBytes{half, half, h * kBlockTokens * 8};
    return GKV_OK;
  case GKV_KV_FP8_BLOCK:
    *out = BlockBytes{half, half, h * 8};
    return GKV_OK;
  default:
    return GKV_ERR_ARG;
  }
}

int copy_blocks(hipStream_t stream, const gkv_cache_view *views, int32_t n_views, int32_t n_pairs,
                const int32_t *src, const int32_t *dst, int stride, const int2 *host_pairs,
                uint32_t *dev_err) {
  // (as many layers a launch as its grid takes; more pairs than that in several launches)
  const int most = std::min(n_pairs, kCopyGrid);
  const int views_at_once = std::min(kCopyViews, kCopyGrid / most);
  for (int v0 = 0; v0 < n_views; v0 += views_at_once) {
    CopyArgs a{};
    a.n_layers = std::min(views_at_once, n_views - v0);
    a.stride = stride;
    a.dev_err = dev_err;
    for (int i = 0; i < a.n_layers; i++) {
      const gkv_cache_view &c = views[v0 + i];
      BlockBytes b;
      const int st = block_bytes(c.n_kv_heads, c.v_format, &b);
      if (st != GKV_OK)
        return st;
      a.layer[i] = CopyLayer{(char *)c.k,         (char *)c.v,         (char *)c.v_scale,
                             (uint32_t)b.k,       (uint32_t)b.v,       (uint32_t)b.s,
                             c.num_blocks};
    }
    for (int64_t p0 = 0; p0 < n_pairs; p0 += most) {
      a.n_pairs = (int)std::min<int64_t>(most, n_pairs - p0);
      a.src = src ? src + p0 * stride : nullptr;
      a.dst = dst ? dst + p0 * stride : nullptr;
      const int items = a.n_layers * a.n_pairs;
      a.parts = items <= kCopySpread / kCopyParts ? kCopyParts : 1;
      const dim3 grid((unsigned)(items * a.parts)), block(kCopyThreads);
      if (host_pairs) {
        InlinePairs in{};
        std::copy(host_pairs, host_pairs + n_pairs, in.p);
        hipLaunchKernelGGL((copy_blocks_kernel<InlinePairs>), grid, block, 0, stream, a, in);
      } else {
        hipLaunchKernelGGL((copy_blocks_kernel<NoPairs>), grid, block, 0, stream, a, NoPairs{});
      }
      const int st = launch_status("copy_blocks_kernel");
      if (st != GKV_OK)
        return st;
    }
  }
  return GKV_OK;
}

} // namespace gkv

extern "C" int gkv_copy_blocks(void *stream, const gkv_cache_view *views, int32_t n_views,
                               int32_t n_pairs, const int32_t *src, const int32_t *dst,
                               uint32_t *dev_err) {
  using namespace gkv;
  if (n_views < 0 || n_pairs < 0 || (n_views > 0 && !views) ||
      (n_views > 0 && n_pairs > 0 && (!src || !dst)))
    return GKV_ERR_ARG;
  for (int i = 0; i < n_views; i++) {
    const gkv_cache_view &c = views[i];
    BlockBytes b;
    if (!c.k || !c.v || c.num_blocks <= 0 || c.n_kv_heads <= 0 || c.n_kv_heads > 65536 ||
        block_bytes(c.n_kv_heads, c.v_format, &b) != GKV_OK || (b.s > 0 && !c.v_scale))
      return GKV_ERR_ARG;
    if (((uintptr_t)c.k | (uintptr_t)c.v) % 16 != 0 || (uintptr_t)c.v_scale % 8 != 0)
      return GKV_ERR_ARG; // 16-byte pieces of K and V, 8-byte pieces of the scales
  }
  if (n_views == 0 || n_pairs == 0)
    return GKV_OK;
  return copy_blocks((hipStream_t)stream, views, n_views, n_pairs, src, dst, 1, nullptr, dev_err);
}
