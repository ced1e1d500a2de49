// Append by whole blocks: RoPE on K, then bf16, or e4m3 codes with one scale per
// block of 16 tokens and kv head, into a cache that may keep first tokens before
// a ring.
//
// The rows of a sequence are consecutive positions, so that the unit of work is
// a block, not a row: one wave takes one (sequence, block, kv head), finds the
// largest |k| and |v| of the block's new tokens, and writes the block once. The
// block's scale is the larger of the one that it has (if the call continues
// it) and the one that the new tokens need; when it grows, the wave moves the older
// codes to it: code' = e4m3(value(code) * s / s'), an exponent shift, which is
// exact unless the result is subnormal.
//
// Lane (kg, t) = (lane / 16, lane % 16) rotates dims 8kg .. 8kg+7 and
// 32+8kg .. +7 of token t and holds their codes as the 16 bytes at lane * 16 of
// the K block (bf16: 16 bytes of each half). V is read by whole rows and goes
// through LDS, from which lane (kg, c) takes tokens 4kg .. 4kg+3 of dims c + 16 n, 16
// contiguous bytes of the V block (bf16: of each half). Every store to the cache
// is 16 bytes a lane, 1 KB a wave, nontemporal: nothing here reads it again
// (prompts 28.9 -> 27.3 us). The angles and the table are those of kv_append.hip,
// the rounding of the rotation too.
//
// Prompts are bound by HBM: 64 of 64 .. 512 rows, 8 kv heads, block scales and
// packed rows, 132 MB in 27.3 us, 4.8 TB/s; bf16, 151 MB, a call 26.6 us, and 512 one-token
// sequences 6.9 (block scales 25.3 and 8.1 in the same run). (V read by 16 dims a lane took four
// times the lines a load: with 8 waves a workgroup 36 us.) A step is bound by latency, the
// lengths, then the table and the angles, then the block: 512 sequences that begin blocks 8.2
// us, of which the launch 2.4, the loads 1.3, the codes 1.5, the stores 2.8.
// The loads of a step's rows and of the table entry therefore go out before
// anything that waits.
#include "kept.hpp"

#include <algorithm>
#include <type_traits>

namespace gkv {

struct KeptAppendArgs {
  const float *qkv;
  int64_t row_stride;
  int n_q_heads, n_kv_heads, max_rows;
  const float *cos_tab, *sin_tab;
  const int32_t *cu, *seq_lens; // cu NULL: one row per sequence
  uint16_t *kc, *vc;            // NULL: packed rows only
  float *scales;
  const int32_t *table;
  int table_stride, num_blocks;
  KeptRow row;
  uint16_t *k_pack, *v_pack;
  uint32_t *dev_err;
};

constexpr int kAppendWaves = 4; // kv heads per workgroup, a wave each
constexpr int kStageRow = kHeadDim + 4; // floats per token in LDS: the transposed reads hit 64 banks

// Maximum over the wave: pairs, quads, half rows and rows of 16 through DPP, then
// rows 0 <-> 1, 2 <-> 3 and the halves, no LDS trip.
__device__ __forceinline__ float wave_max(float x) {
  auto dpp = [](float v, auto c) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), decltype(c)::value, 0xf, 0xf, false));
  };
  x = fmaxf(x, dpp(x, std::integral_constant<int, 0xb1>{}));
  x = fmaxf(x, dpp(x, std::integral_constant<int, 0x4e>{}));
  x = fmaxf(x, dpp(x, std::integral_constant<int, 0x141>{}));
  x = fmaxf(x, dpp(x, std::integral_constant<int, 0x140>{}));
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}

// |x|, 0 where x is not finite (such a value saturates or becomes NaN by
// itself; it must not take the block's other tokens' resolution).
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.0f;
}

// Four e4m3 codes of x * inv, saturated; a NaN stays one.
__device__ __forceinline__ uint32_t block_codes(float x0, float x1, float x2, float x3,
                                                float inv) {
  auto c = [inv](float x) {
    const float y = x * inv;
    return y > 448.0f ? 448.0f : y < -448.0f ? -448.0f : y;
  };
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(c(x0), c(x1), 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c(x2), c(x3), w, true);
}

// The same four codes under a scale `ratio` times smaller (ratio <= 1).
__device__ __forceinline__ uint32_t move_codes(uint32_t w, float ratio) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  return block_codes(a[0], a[1], b[0], b[1], ratio);
}

// BLK: e4m3 with block scales, else bf16.
template <bool BLK>
__global__ __launch_bounds__(64 * kAppendWaves) void kept_append_kernel(KeptAppendArgs a) {
  constexpr int D = kHeadDim, HALF = kHeadDim / 2;
  __shared__ __attribute__((aligned(16))) float s_v[kAppendWaves][kBlockTokens * kStageRow];
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int b = blockIdx.y, g = blockIdx.z * kAppendWaves + wave, t = lane & 15, kg = lane >> 4;
  if (g >= a.n_kv_heads)
    return;
  const int row0 = a.cu ? a.cu[b] : b, n = a.cu ? a.cu[b + 1] - row0 : 1;
  const int L = a.seq_lens[b], start = L - n; // the rows are positions start .. L - 1

  // The new tokens' rows of head g: K dims 8kg .. +7 and 32+8kg .. +7 of token t, V
  // dims 4t .. +3 of tokens 4i + kg. In a call of one row per sequence every lane
  // reads that row, whose address waits for no length.
  f32x4 x[4], y[4];
  int p0 = 0, n_old = 0, n_end = 0;
  auto load_rows = [&] {
    const float *base = a.qkv + (int64_t)(a.n_q_heads + g) * D;
    const int64_t row_p0 = (int64_t)row0 + (p0 - start);
#pragma unroll
    for (int i = 0; i < 4; i++)
      x[i] = y[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (!a.cu || (t >= n_old && t < n_end)) {
      const f32x4 *kp = (const f32x4 *)(base + (a.cu ? row_p0 + t : b) * a.row_stride + 8 * kg);
      x[0] = kp[0];
      x[1] = kp[1];
      x[2] = kp[HALF / 4];
      x[3] = kp[HALF / 4 + 1];
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int tok = 4 * i + kg;
      if (!a.cu || (tok >= n_old && tok < n_end))
        y[i] = *(const f32x4 *)(base + (a.cu ? row_p0 + tok : b) * a.row_stride +
                                a.n_kv_heads * D + 4 * t);
    }
  };
  if (!a.cu)
    load_rows();

  if (n <= 0)
    return;
  if (n > a.max_rows && blockIdx.x == 0 && threadIdx.x == 0 && a.dev_err)
    atomicOr(a.dev_err, GKV_DEVERR_LENGTH); // (the grid covers max_rows)
  const int blk = max(start, 0) / kBlockTokens + blockIdx.x;
  p0 = blk * kBlockTokens;
  if (p0 >= L)
    return;
  // Where the block stands: its table entry's load goes out here, beside the rows',
  // and is looked at behind them. A block that a later one of this call replaces
  // in the ring is not stored.
  const int last = (L - 1) / kBlockTokens;
  const bool later = a.row.ring_blocks > 0 && blk >= a.row.kept_blocks &&
                     blk + a.row.ring_blocks <= last;
  const int entry = kept_entry(a.row, blk);
  int phys = 0;
  if (a.kc && entry < a.table_stride)
    phys = a.table[(int64_t)b * a.table_stride + entry];
  n_old = max(min(start - p0, kBlockTokens), 0); // tokens the block holds already
  n_end = min(L - p0, kBlockTokens);             // ... and after the call
  const bool is_new = t >= n_old && t < n_end;
  if (a.cu)
    load_rows();
  // The angles, one token a lane (of a full row's last position past its
  // capacity: the caller's tables need not reach further).
  f32x4 c[2], s[2];
  {
    const f32x4 zero{0.0f, 0.0f, 0.0f, 0.0f};
    c[0] = c[1] = s[0] = s[1] = zero;
    const int64_t cap = kept_capacity(a.table_stride, a.row.ring_blocks);
    const int pos = (int)min((int64_t)(p0 + t), a.kc ? cap - 1 : (int64_t)p0 + t);
    if (is_new) {
      const f32x4 *cp = (const f32x4 *)(a.cos_tab + (int64_t)pos * HALF + 8 * kg);
      const f32x4 *sp = (const f32x4 *)(a.sin_tab + (int64_t)pos * HALF + 8 * kg);
      c[0] = cp[0];
      c[1] = cp[1];
      s[0] = sp[0];
      s[1] = sp[1];
    }
  }
  bool store = a.kc != nullptr && !later;
  if (store && entry >= a.table_stride) {
    if (threadIdx.x == 0 && a.dev_err)
      atomicOr(a.dev_err, GKV_DEVERR_LENGTH);
    store = false;
  }
  if (store && (uint32_t)phys >= (uint32_t)a.num_blocks) {
    if (threadIdx.x == 0 && a.dev_err)
      atomicOr(a.dev_err, GKV_DEVERR_BLOCK_ID);
    store = false;
  }
  const int64_t base = store ? (int64_t)phys * a.n_kv_heads : 0;
  float *sv = s_v[wave];
  const int v_at = BLK ? (t * 4 + kg) * 16 : lane * 16; // this lane's piece of a V block

  if (!a.cu) { // the row is one token's
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int tok = 4 * i + kg;
      if (!is_new)
        x[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (tok < n_old || tok >= n_end)
        y[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
  }
  // the codes and scales that the block has
  u32x4 k_was{0, 0, 0, 0}, v_was{0, 0, 0, 0}, v_was2{0, 0, 0, 0};
  f32x2 sc_was{0.0f, 0.0f};
  const int64_t hb = base + g; // the head's block
  uint8_t *kd = (uint8_t *)a.kc + hb * (BLK ? 1024 : 2048);
  uint8_t *vd = (uint8_t *)a.vc + hb * (BLK ? 1024 : 2048);
  if (store && n_old > 0) {
    if (BLK) {
      sc_was = *(const f32x2 *)(a.scales + 2 * hb);
      k_was = *(const u32x4 *)(kd + lane * 16);
    }
    v_was = *(const u32x4 *)(vd + v_at);
    if (!BLK)
      v_was2 = *(const u32x4 *)(vd + 1024 + lane * 16);
  }
  float f1[8], f2[8];
  float ka = 0.0f, va = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const float x1 = x[i / 4][i % 4], x2 = x[2 + i / 4][i % 4];
    const float cc = c[i / 4][i % 4], ss = s[i / 4][i % 4];
    f1[i] = rope_first(x1, x2, cc, ss);
    f2[i] = rope_second(x1, x2, cc, ss);
    if (BLK) {
      ka = fmaxf(ka, fmaxf(finite_abs(f1[i]), finite_abs(f2[i])));
      va = fmaxf(va, fmaxf(finite_abs(y[i / 2][2 * (i % 2)]), finite_abs(y[i / 2][2 * (i % 2) + 1])));
    }
  }
  if (a.k_pack && is_new) {
    uint16_t *o = a.k_pack + ((row0 + (int64_t)(p0 + t - start)) * a.n_kv_heads + g) * D;
    *(u32x4 *)(o + 8 * kg) = round8(f1);
    *(u32x4 *)(o + HALF + 8 * kg) = round8(f2);
  }
  if (a.v_pack) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int tok = 4 * i + kg;
      if (tok >= n_old && tok < n_end)
        *(u32x2 *)(a.v_pack + ((row0 + (int64_t)(p0 + tok - start)) * a.n_kv_heads + g) * D + 4 * t) =
            u32x2{f32x2_to_bf16_rne(y[i][0], y[i][1]), f32x2_to_bf16_rne(y[i][2], y[i][3])};
    }
  }
  if (!store)
    return;
  // V by columns: tokens 4kg + r of dims t + 16 n (this wave's own LDS, whose
  // accesses stay in order)
#pragma unroll
  for (int i = 0; i < 4; i++)
    *(f32x4 *)(sv + (4 * i + kg) * kStageRow + 4 * t) = y[i];
  __builtin_amdgcn_wave_barrier();
  float v[4][4];
#pragma unroll
  for (int nn = 0; nn < 4; nn++)
#pragma unroll
    for (int q = 0; q < 4; q++)
      v[nn][q] = sv[(4 * kg + q) * kStageRow + t + 16 * nn];
  __builtin_amdgcn_wave_barrier();
  uint32_t fresh = 0; // a byte of ones per token of this lane's V piece that is new
#pragma unroll
  for (int q = 0; q < 4; q++)
    fresh |= 4 * kg + q >= n_old && 4 * kg + q < n_end ? 0xffu << (8 * q) : 0u;

  if constexpr (BLK) {
    ka = wave_max(ka);
    va = wave_max(va);
    const float sk = fmaxf(sc_was[0], block_scale(ka)), sv2 = fmaxf(sc_was[1], block_scale(va));
    // (scale 0: only zeros, and what is not finite, which saturates or stays a NaN)
    const float ik = sk > 0.0f ? 1.0f / sk : 1.0f, iv = sv2 > 0.0f ? 1.0f / sv2 : 1.0f;
    const bool grow_k = n_old > 0 && sk != sc_was[0], grow_v = n_old > 0 && sv2 != sc_was[1];
    // K: a new token's codes; an older one's, moved, if the scale grew; zeros
    // behind the tokens of a block that this call begins
    if (is_new || n_old == 0 || (grow_k && t < n_old)) {
      u32x4 w{0, 0, 0, 0};
      if (is_new) {
        w = u32x4{block_codes(f1[0], f1[1], f1[2], f1[3], ik),
                  block_codes(f1[4], f1[5], f1[6], f1[7], ik),
                  block_codes(f2[0], f2[1], f2[2], f2[3], ik),
                  block_codes(f2[4], f2[5], f2[6], f2[7], ik)};
      } else if (n_old > 0) {
        const float ratio = sc_was[0] * ik;
#pragma unroll
        for (int i = 0; i < 4; i++)
          w[i] = move_codes(k_was[i], ratio);
      }
      __builtin_nontemporal_store(w, (u32x4 *)(kd + lane * 16));
    }
    if (fresh != 0 || n_old == 0 || (grow_v && 4 * kg < n_old)) {
      uint32_t older = 0;
#pragma unroll
      for (int q = 0; q < 4; q++)
        older |= 4 * kg + q < n_old ? 0xffu << (8 * q) : 0u;
      const float ratio = sc_was[1] * iv;
      u32x4 w;
#pragma unroll
      for (int nn = 0; nn < 4; nn++) {
        uint32_t was = v_was[nn];
        if (grow_v)
          was = (move_codes(was, ratio) & older) | (was & ~older);
        w[nn] = (block_codes(v[nn][0], v[nn][1], v[nn][2], v[nn][3], iv) & fresh) | (was & ~fresh);
      }
      __builtin_nontemporal_store(w, (u32x4 *)(vd + v_at));
    }
    if (lane == 0)
      *(f32x2 *)(a.scales + 2 * hb) = f32x2{sk, sv2};
  } else {
    if (is_new || n_old == 0) {
      __builtin_nontemporal_store(round8(f1), (u32x4 *)(kd + lane * 16));
      __builtin_nontemporal_store(round8(f2), (u32x4 *)(kd + 1024 + lane * 16));
    }
    if (fresh != 0 || n_old == 0) {
      const uint32_t m0 = (fresh & 0xffu ? 0xffffu : 0u) | (fresh & 0xff00u ? 0xffff0000u : 0u);
      const uint32_t m1 =
          (fresh & 0xff0000u ? 0xffffu : 0u) | (fresh & 0xff000000u ? 0xffff0000u : 0u);
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const u32x4 was = h ? v_was2 : v_was;
        u32x4 w;
#pragma unroll
        for (int k = 0; k < 2; k++) { // dims t + 32 h and t + 32 h + 16
          const float *f = v[2 * h + k];
          w[2 * k] = (f32x2_to_bf16_rne(f[0], f[1]) & m0) | (was[2 * k] & ~m0);
          w[2 * k + 1] = (f32x2_to_bf16_rne(f[2], f[3]) & m1) | (was[2 * k + 1] & ~m1);
        }
        __builtin_nontemporal_store(w, (u32x4 *)(vd + h * 1024 + lane * 16));
      }
    }
  }
}

} // namespace gkv

extern "C" int gkv_kept_append(void *stream, int32_t B, const int32_t *cu_seqlens,
                               const int32_t *seq_lens, int32_t max_rows, const float *qkv,
                               int64_t row_stride, int32_t n_q_heads, const float *cos_tab,
                               const float *sin_tab, gkv_cache_view cache, int32_t kept,
                               int32_t window, void *k_pack, void *v_pack, uint32_t *dev_err) {
  using namespace gkv;
  if (B < 0 || max_rows < 0 || !seq_lens || !qkv || !cos_tab || !sin_tab || n_q_heads <= 0)
    return GKV_ERR_ARG;
  const bool to_cache = cache.k != nullptr || cache.v != nullptr;
  const int st = kept_check(cache, kept, window, to_cache);
  if (st != GKV_OK)
    return st;
  if (n_q_heads % cache.n_kv_heads != 0 ||
      row_stride < ((int64_t)n_q_heads + 2 * (int64_t)cache.n_kv_heads) * kHeadDim)
    return GKV_ERR_ARG;
  // 16-byte vector loads and stores
  if (row_stride % 4 != 0 ||
      ((uintptr_t)qkv | (uintptr_t)cos_tab | (uintptr_t)sin_tab | (uintptr_t)k_pack |
       (uintptr_t)v_pack) % 16 != 0)
    return GKV_ERR_ARG;
  if (B > 65535)
    return GKV_ERR_UNSUPPORTED; // a grid row per sequence
  if (cu_seqlens == nullptr && max_rows > 1)
    return GKV_ERR_ARG;
  // blocks that max_rows consecutive positions can touch
  const int64_t blocks = (max_rows + (int64_t)kBlockTokens - 2) / kBlockTokens + 1;
  if (!grid_fits(blocks, 64 * kAppendWaves))
    return GKV_ERR_UNSUPPORTED;
  if (B == 0 || max_rows == 0 || (!to_cache && !k_pack && !v_pack))
    return GKV_OK;
  KeptAppendArgs a;
  a.qkv = qkv;
  a.row_stride = row_stride;
  a.n_q_heads = n_q_heads;
  a.n_kv_heads = cache.n_kv_heads;
  a.max_rows = max_rows;
  a.cos_tab = cos_tab;
  a.sin_tab = sin_tab;
  a.cu = cu_seqlens;
  a.seq_lens = seq_lens;
  a.kc = to_cache ? (uint16_t *)cache.k : nullptr;
  a.vc = to_cache ? (uint16_t *)cache.v : nullptr;
  a.scales = (float *)cache.v_scale;
  a.table = cache.block_table;
  a.table_stride = cache.table_stride;
  a.num_blocks = cache.num_blocks;
  a.row = KeptRow{kept / kBlockTokens, cache.ring / kBlockTokens};
  a.k_pack = (uint16_t *)k_pack;
  a.v_pack = (uint16_t *)v_pack;
  a.dev_err = dev_err;
  const int waves = std::min(kAppendWaves, a.n_kv_heads);
  const dim3 grid((unsigned)blocks, B, (unsigned)((a.n_kv_heads + waves - 1) / waves));
  const dim3 block(64 * waves);
  if (to_cache && cache.v_format == GKV_KV_FP8_BLOCK)
    hipLaunchKernelGGL((kept_append_kernel<true>), grid, block, 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL((kept_append_kernel<false>), grid, block, 0, (hipStream_t)stream, a);
  return launch_status("kept_append_kernel");
}
