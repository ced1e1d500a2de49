// What the gkv_kept_* entry points share: where a position's block stands in a
// sequence's table row, which positions a query sees, and the block format's
// scales.
//
// Position t is seen from position p iff t <= p and (t < kept or t > p - window);
// window 0: every t <= p. kept and window are multiples of 16. Logical block j
// (positions 16 j .. 16 j + 15) is entry j of the table row, or, on a ring of
// window + 16 slots, entry j of the kept blocks and behind them entry
// kept / 16 + (j - kept / 16) % (window / 16 + 1). The ring holds one block more
// than the window, so that when a token begins a block none of the block's former
// tokens is seen any more: the block's scale can start over, and a masked
// token is never overwritten while its block is read.
#pragma once

#include "kv_append.hpp"

namespace gkv {

struct KeptRow {
  int kept_blocks; // kept / 16
  int ring_blocks; // blocks of the ring (0: every position's block in the row)
};

// Table entry of logical block j.
__host__ __device__ __forceinline__ int kept_entry(const KeptRow &r, int j) {
  return r.ring_blocks == 0 || j < r.kept_blocks
             ? j
             : r.kept_blocks + (int)((uint32_t)(j - r.kept_blocks) % (uint32_t)r.ring_blocks);
}

// Checks of the arguments that say how the cache is laid out, the same for
// every entry point. need_cache: the call reads or writes the paged cache.
inline int kept_check(const gkv_cache_view &c, int32_t kept, int32_t window, bool need_cache) {
  if (c.n_kv_heads <= 0 || kept < 0 || window < 0 || c.ring < 0)
    return GKV_ERR_ARG;
  if (kept % kBlockTokens != 0 || window % kBlockTokens != 0)
    return GKV_ERR_UNSUPPORTED;
  if (!need_cache)
    return GKV_OK;
  if (c.v_format == GKV_V_INT8 || c.v_format == GKV_KV_FP8)
    return GKV_ERR_UNSUPPORTED;
  if (c.v_format != GKV_V_BF16 && c.v_format != GKV_KV_FP8_BLOCK)
    return GKV_ERR_ARG;
  if (!c.k || !c.v || !c.block_table || c.table_stride <= 0 || c.num_blocks <= 0 ||
      (c.v_format == GKV_KV_FP8_BLOCK && !c.v_scale))
    return GKV_ERR_ARG;
  if (((uintptr_t)c.k | (uintptr_t)c.v) % 16 != 0 || (uintptr_t)c.v_scale % 8 != 0 ||
      (uintptr_t)c.block_table % 4 != 0)
    return GKV_ERR_ARG; // 16-byte pieces of K and V, 8-byte pairs of scales
  if (c.ring > 0 && (window == 0 || c.ring != (int64_t)window + kBlockTokens ||
                     (int64_t)c.table_stride * kBlockTokens < (int64_t)kept + c.ring))
    return GKV_ERR_ARG; // a ring of window + 16 slots behind the kept blocks
  return GKV_OK;
}

// Positions a full table row can hold (a ring holds any).
__host__ __device__ __forceinline__ int64_t kept_capacity(int table_stride, int ring_blocks) {
  return ring_blocks > 0 ? (int64_t)1 << 31 : (int64_t)table_stride * kBlockTokens;
}

// The block format's scale for values up to amax (finite): the smallest power
// of two s with amax <= 448 s, from the bits (448 = 1.75 * 2^8); 0 for amax 0. A
// power of two costs e4m3 no precision (the codes keep their 3 mantissa bits
// whatever the scale), makes value * (1 / s) exact, and a later, larger scale
// moves the older codes' exponents only.
__host__ __device__ __forceinline__ float block_scale(float amax) {
  union {
    float f;
    uint32_t u;
  } x;
  x.f = amax;
  if (amax == 0.0f)
    return 0.0f;
  int e = (int)(x.u >> 23) - 8 + ((x.u & 0x7fffffu) > 0x600000u ? 1 : 0);
  x.u = (uint32_t)(e < 1 ? 1 : e) << 23;
  return x.f;
}

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Four e4m3 codes -> four fp16 of code * scale, scale a power of two (1: exact).
__device__ __forceinline__ u32x2 codes_to_f16(uint32_t w, float scale = 1.0f) {
  const f16x2 a = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, false));
  const f16x2 b = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, true));
  return u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
}

} // namespace gkv
