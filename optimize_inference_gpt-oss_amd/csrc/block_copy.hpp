// Copies of whole cache blocks (block_copy.hip), shared by gkv_copy_blocks and
// the pool's fork, trim and compaction.
#pragma once

#include "gkv_device.hpp"

namespace gkv {

constexpr int kInlinePairs = 128; // pairs that travel as kernel arguments

// Bytes of one block of one layer: K, V and scales.
struct BlockBytes {
  int64_t k, v, s;
};
int block_bytes(int n_kv_heads, int v_format, BlockBytes *out);

// Copies block src[i * stride] to dst[i * stride] in every view (checked by
// the caller), the ids in device memory, or, with host_pairs (at most
// kInlinePairs of {src, dst}), in the kernel's arguments.
int copy_blocks(hipStream_t stream, const gkv_cache_view *views, int32_t n_views, int32_t n_pairs,
                const int32_t *src, const int32_t *dst, int stride, const int2 *host_pairs,
                uint32_t *dev_err);

} // namespace gkv
