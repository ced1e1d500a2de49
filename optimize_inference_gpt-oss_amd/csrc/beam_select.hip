// Beam search's choice: for every request the n best of its beams' continuations.
//
// A continuation of beam b by token t scores cum[b] + x[b][t] - log sum_v exp x[b][v]. The
// logits are read once: a wave takes a run of a row, keeps the row's running maximum and sum
// per lane, and its n best so far in one register across its lanes, sorted. Inside a row the
// order is that of the logits, so nothing but their values is compared until the rows meet;
// scores are formed and compared in 64 bits (two beams' scores differ by as little as
// their sums' last bits).
#include "gkv_device.hpp"

#include <algorithm>

namespace gkv {

constexpr int kBeamMost = 64;      // candidates per request, at most: one a lane
constexpr int kBeamThreads = 256;  // four waves of a row's part
constexpr int kBeamWaves = kBeamThreads / 64;
constexpr int kMergeWaves = 8;
constexpr float kFloatMax = 3.402823466e38f;

struct BeamArgs {
  const void *x;
  int64_t stride;
  const float *cum;
  const int32_t *done;
  int R, K, V, n, eos;
  int parts;        // workgroups per row
  float2 *ml;       // [rows][parts] maximum, sum of exp2((x - maximum) log2 e)
  float *best;      // [rows][parts][n] logits, best first
  int32_t *token;   // and their tokens; -1: there is none
  float *scores;
  int32_t *parents, *tokens, *done_out;
  uint32_t *dev_err;
};

// A value's place in the order of floats, as an unsigned number; 0 is below every value.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// A logit as it counts: NaN as -inf, +inf as the largest number.
__device__ __forceinline__ float plain_logit(float x) {
  return x != x ? -INFINITY : fminf(x, kFloatMax);
}

// The n best of what a wave has met, entry i in lane i, best first; equal ones in the order
// in which they came.
struct Best {
  float x;
  int token;      // -1: no entry
  float low;      // the n-th (-inf while there are fewer)
  bool full;
};

__device__ __forceinline__ void insert(Best &b, float x, int token, int n) {
  const int lane = threadIdx.x & 63;
  const uint64_t before = __ballot(b.token >= 0 && b.x >= x);
  const int at = __popcll(before);
  const float ux = __shfl_up(b.x, 1, 64);
  const int ut = __shfl_up(b.token, 1, 64);
  if (lane == at) {
    b.x = x;
    b.token = token;
  } else if (lane > at) {
    b.x = ux;
    b.token = ut;
  }
  b.low = __shfl(b.x, n - 1, 64);
  b.full = __shfl(b.token, n - 1, 64) >= 0;
}

// The row's 16-byte granule i (aligned down from the row's start, off elements before it) as
// fp32; elements outside the row are -inf and not read.
template <bool BF>
struct Granule {
  static constexpr int N = BF ? 8 : 4;
  float v[N];
};
template <bool BF>
__device__ __forceinline__ void load_granule(Granule<BF> &g, const char *base, int64_t i, int64_t off,
                                             int64_t V) {
  constexpr int N = Granule<BF>::N;
  const int64_t e = i * N - off;
  if (e >= 0 && e + N <= V) {
    const u32x4 w = __builtin_nontemporal_load((const u32x4 *)base + i);
#pragma unroll
    for (int j = 0; j < N; j++)
      g.v[j] = BF ? __uint_as_float(j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16)
                  : __uint_as_float(w[j % 4]);
  } else {
#pragma unroll
    for (int j = 0; j < N; j++) {
      g.v[j] = -INFINITY;
      if (e + j >= 0 && e + j < V)
        g.v[j] = BF ? bf16_to_f32(((const uint16_t *)base)[i * N + j])
                    : ((const float *)base)[i * N + j];
    }
  }
}

template <bool BF>
__global__ __launch_bounds__(kBeamThreads) void beam_rows_kernel(BeamArgs a) {
  constexpr int N = Granule<BF>::N, U = 16 / N; // granules a lane takes in one go
  __shared__ float s_x[kBeamWaves][kBeamMost];
  __shared__ int s_t[kBeamWaves][kBeamMost];
  __shared__ float2 s_ml[kBeamWaves];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int row = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  // (a row that is finished, or that no score can reach, is not read)
  const float cum = a.cum[row];
  if ((a.done && a.done[row] != 0) || !(cum > -INFINITY))
    return;
  const char *start = (const char *)a.x + (int64_t)row * a.stride * (BF ? 2 : 4);
  const int64_t off = ((uintptr_t)start & 15) / (BF ? 2 : 4);
  const char *base = (const char *)((uintptr_t)start & ~(uintptr_t)15);
  // this wave's tiles of 64 U granules, in order
  const int64_t granules = (off + a.V + N - 1) / N, tiles = (granules + 64 * U - 1) / (64 * U);
  const int64_t w = (int64_t)part * kBeamWaves + wave, n_waves = (int64_t)a.parts * kBeamWaves;
  const int64_t t0 = w * tiles / n_waves, t1 = (w + 1) * tiles / n_waves;

  Best best{-INFINITY, -1, -INFINITY, false};
  float m = -kFloatMax, l = 0.0f;
  bool odd = false; // a NaN or +inf was met
  Granule<BF> g[U];
#pragma unroll
  for (int u = 0; u < U; u++)
    load_granule<BF>(g[u], base, t0 < t1 ? t0 * 64 * U + u * 64 + lane : granules, off, a.V);
  for (int64_t t = t0; t < t1; t++) {
    Granule<BF> c[U];
#pragma unroll
    for (int u = 0; u < U; u++)
      c[u] = g[u];
    if (t + 1 < t1)
#pragma unroll
      for (int u = 0; u < U; u++)
        load_granule<BF>(g[u], base, (t + 1) * 64 * U + u * 64 + lane, off, a.V);
    float mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int j = 0; j < N; j++) {
        odd |= !(c[u].v[j] <= kFloatMax);
        c[u].v[j] = plain_logit(c[u].v[j]);
        mx = fmaxf(mx, c[u].v[j]);
      }
    const float mn = fmaxf(m, mx);
    l *= __builtin_amdgcn_exp2f((m - mn) * kLog2e);
    m = mn;
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int j = 0; j < N; j++)
        l += __builtin_amdgcn_exp2f((c[u].v[j] - m) * kLog2e);
    if (best.full && !__any(mx > best.low))
      continue;
    // in the order of the tokens: granule after granule, lane after lane
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int64_t e0 = (t * 64 * U + u * 64 + lane) * N - off;
      uint32_t mask = 0;
#pragma unroll
      for (int j = 0; j < N; j++)
        if (e0 + j >= 0 && e0 + j < a.V && (!best.full || c[u].v[j] > best.low))
          mask |= 1u << j;
      for (;;) {
        const uint64_t who = __ballot(mask != 0);
        if (who == 0)
          break;
        const int from = __ffsll((unsigned long long)who) - 1;
        const int j = __shfl(__ffs(mask) - 1, from, 64);
        float x = c[u].v[0];
#pragma unroll
        for (int k = 1; k < N; k++)
          x = j == k ? c[u].v[k] : x;
        x = __shfl(x, from, 64);
        const int64_t e = __shfl(e0, from, 64) + j;
        if (lane == from)
          mask &= mask - 1;
        if (!best.full || x > best.low) {
          insert(best, x, (int)e, a.n);
          // (what no longer gets in is dropped at once)
#pragma unroll
          for (int k = 0; k < N; k++)
            if (best.full && !(c[u].v[k] > best.low))
              mask &= ~(1u << k);
        }
      }
    }
  }
  if (__any(odd) && lane == 0 && a.dev_err)
    atomicOr(a.dev_err, GKV_DEVERR_RANGE);
  // the lanes' sums, then the waves'
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const float m2 = __shfl_xor(m, o), l2 = __shfl_xor(l, o), mn = fmaxf(m, m2);
    l = l * __builtin_amdgcn_exp2f((m - mn) * kLog2e) + l2 * __builtin_amdgcn_exp2f((m2 - mn) * kLog2e);
    m = mn;
  }
  if (lane == 0)
    s_ml[wave] = float2{m, l};
  s_x[wave][lane] = best.x;
  s_t[wave][lane] = lane < a.n ? best.token : -1;
  __syncthreads();
  const int64_t at = (int64_t)row * a.parts + part;
  if (threadIdx.x == 0) {
    for (int k = 1; k < kBeamWaves; k++) {
      const float mn = fmaxf(m, s_ml[k].x);
      l = l * __builtin_amdgcn_exp2f((m - mn) * kLog2e) +
          s_ml[k].y * __builtin_amdgcn_exp2f((s_ml[k].x - mn) * kLog2e);
      m = mn;
    }
    a.ml[at] = float2{m, l};
  }
  // an entry's place among all the waves': those above it, and equal ones of lower tokens
  const float x = s_x[wave][lane];
  const int token = s_t[wave][lane];
  int place = 0, entries = 0;
  for (int k = 0; k < kBeamWaves; k++)
    for (int i = 0; i < a.n; i++) {
      const float y = s_x[k][i];
      const int o = s_t[k][i];
      entries += o >= 0;
      place += o >= 0 && (y > x || (y == x && o < token));
    }
  if (token >= 0 && place < a.n) {
    a.best[at * a.n + place] = x;
    a.token[at * a.n + place] = token;
  }
  for (int i = entries + threadIdx.x; i < a.n; i += kBeamThreads)
    a.token[at * a.n + i] = -1;
}

// One candidate: its score and flat index beam * V + token (-1: none).
struct Candidate {
  double s;
  int64_t at;
};
__device__ __forceinline__ bool beats(double s, int64_t at, double s2, int64_t at2) {
  return at >= 0 && (at2 < 0 || s > s2 || (s == s2 && at < at2));
}

__device__ __forceinline__ void insert(Candidate &b, double s, int64_t at) {
  const int lane = threadIdx.x & 63;
  const int place = __popcll(__ballot(beats(b.s, b.at, s, at)));
  const double us = __shfl_up(b.s, 1, 64);
  const int64_t ua = __shfl_up(b.at, 1, 64);
  if (lane == place) {
    b.s = s;
    b.at = at;
  } else if (lane > place) {
    b.s = us;
    b.at = ua;
  }
}

// A workgroup per request: the rows' sums, then the best of their best.
__global__ __launch_bounds__(64 * kMergeWaves) void beam_merge_kernel(BeamArgs a) {
  __shared__ double s_lse[kBeamMost];
  __shared__ double s_s[kMergeWaves][kBeamMost];
  __shared__ int64_t s_at[kMergeWaves][kBeamMost];
  const int r = blockIdx.x, lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  for (int k = wave; k < a.K; k += kMergeWaves) {
    const int row = r * a.K + k;
    const float cum = a.cum[row];
    if (!(cum <= kFloatMax) && lane == 0 && a.dev_err)
      atomicOr(a.dev_err, GKV_DEVERR_RANGE);
    if ((a.done && a.done[row] != 0) || !(cum > -INFINITY))
      continue;
    float m = -kFloatMax;
    for (int p = lane; p < a.parts; p += 64)
      m = fmaxf(m, a.ml[(int64_t)row * a.parts + p].x);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1)
      m = fmaxf(m, __shfl_xor(m, o));
    double l = 0;
    for (int p = lane; p < a.parts; p += 64) {
      const float2 ml = a.ml[(int64_t)row * a.parts + p];
      l += (double)ml.y * exp2(((double)ml.x - (double)m) * 1.4426950408889634);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1)
      l += __shfl_xor(l, o);
    if (lane == 0) // (a row of -inf alone: every score is -inf)
      s_lse[k] = l > 0 ? (double)m + log(l) : 0.0;
  }
  __syncthreads();
  Candidate b{0.0, -1};
  const int per_row = a.parts * a.n;
  double low = 0;
  int64_t low_at = -1;
  for (int i0 = wave * 64; i0 < a.K * per_row; i0 += 64 * kMergeWaves) {
    const int i = i0 + lane, k = i / per_row, e = i % per_row, row = r * a.K + k;
    double s = 0;
    int64_t at = -1;
    if (k < a.K) {
      const float cum = a.cum[row];
      const double c = cum != cum ? -INFINITY : (double)fminf(cum, kFloatMax);
      if (a.done && a.done[row] != 0) {
        // its one continuation, and tokens that score -inf
        if (e < a.n) {
          const int t = e == 0 ? a.eos : e - 1 < a.eos ? e - 1 : e;
          s = e == 0 ? c : -INFINITY;
          at = t < a.V ? (int64_t)k * a.V + t : -1;
        }
      } else if (!(c > -INFINITY)) {
        if (e < a.n) {
          s = -INFINITY;
          at = (int64_t)k * a.V + e;
        }
      } else {
        const int64_t p = (int64_t)row * per_row + e;
        const int t = a.token[p];
        if (t >= 0) {
          s = c + ((double)a.best[p] - s_lse[k]);
          at = (int64_t)k * a.V + t;
        }
      }
    }
    bool in = beats(s, at, low, low_at);
    for (;;) {
      const uint64_t who = __ballot(in);
      if (who == 0)
        break;
      const int from = __ffsll((unsigned long long)who) - 1;
      const double fs = __shfl(s, from, 64);
      const int64_t fa = __shfl(at, from, 64);
      insert(b, fs, fa);
      low = __shfl(b.s, a.n - 1, 64);
      low_at = __shfl(b.at, a.n - 1, 64);
      in = in && lane != from && beats(s, at, low, low_at);
    }
  }
  s_s[wave][lane] = b.s;
  s_at[wave][lane] = lane < a.n ? b.at : -1;
  __syncthreads();
  if (b.at < 0 || lane >= a.n)
    return;
  int place = 0;
  for (int k = 0; k < kMergeWaves; k++)
    for (int i = 0; i < a.n; i++)
      place += beats(s_s[k][i], s_at[k][i], b.s, b.at);
  if (place < a.n) {
    const int64_t o = (int64_t)r * a.n + place;
    const int row = r * a.K + (int)(b.at / a.V), t = (int)(b.at % a.V);
    a.scores[o] = (float)b.s;
    a.parents[o] = row;
    a.tokens[o] = t;
    if (a.done_out)
      a.done_out[o] = t == a.eos || (a.done && a.done[row] != 0);
  }
}

// Workgroups per row: as many as give every CU eight waves, as long as a wave keeps a tile of
// 1024 logits.
constexpr int kBeamWgs = 512;
static int beam_parts(int64_t rows, int32_t V) {
  const int64_t tiles = ((int64_t)V + 1023) / 1024;
  const int64_t most = std::max<int64_t>(1, tiles / kBeamWaves);
  return (int)std::max<int64_t>(1, std::min<int64_t>(most, kBeamWgs / std::max<int64_t>(rows, 1)));
}

struct BeamWorkspace {
  size_t best, token, total;
};
static BeamWorkspace beam_workspace(int64_t rows, int n) {
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  BeamWorkspace w;
  const size_t pieces = std::max<int64_t>(rows, kBeamWgs); // (what fewer rows need too)
  w.best = up(pieces * sizeof(float2));
  w.token = w.best + up(pieces * n * 4);
  w.total = w.token + pieces * n * 4;
  return w;
}

static bool beam_sizes_ok(int32_t R, int32_t K, int32_t V, int32_t n) {
  return R >= 0 && K > 0 && V > 0 && n > 0 && n <= V && n <= kBeamMost && K <= kBeamMost &&
         (int64_t)R * K < (1 << 23);
}

} // namespace gkv

extern "C" size_t gkv_beam_workspace_bytes(int32_t n_requests, int32_t n_beams, int32_t vocab,
                                           int32_t n_out) {
  using namespace gkv;
  if (!beam_sizes_ok(n_requests, n_beams, vocab, n_out))
    return 0;
  const int64_t rows = (int64_t)n_requests * n_beams;
  return beam_workspace(rows, n_out).total;
}

extern "C" int gkv_beam_select(void *stream, int32_t n_requests, int32_t n_beams, int32_t vocab,
                               const void *logits, int64_t row_stride, int32_t logits_dtype,
                               const float *cum_scores, const int32_t *done, int32_t eos,
                               int32_t n_out, float *scores, int32_t *parents, int32_t *tokens,
                               int32_t *done_out, void *workspace, size_t workspace_bytes,
                               uint32_t *dev_err) {
  using namespace gkv;
  if (n_requests < 0 || n_beams <= 0 || vocab <= 0 || n_out <= 0 || n_out > vocab || !logits ||
      !cum_scores || !scores || !parents || !tokens || row_stride < vocab ||
      (logits_dtype != GKV_F32 && logits_dtype != GKV_BF16) || eos >= vocab || (done && eos < 0))
    return GKV_ERR_ARG;
  const bool bf = logits_dtype == GKV_BF16;
  if ((uintptr_t)logits % (bf ? 2 : 4) != 0 ||
      ((uintptr_t)cum_scores | (uintptr_t)done | (uintptr_t)scores | (uintptr_t)parents |
       (uintptr_t)tokens | (uintptr_t)done_out) % 4 != 0 || (uintptr_t)workspace % 16 != 0)
    return GKV_ERR_ARG;
  if (!beam_sizes_ok(n_requests, n_beams, vocab, n_out))
    return GKV_ERR_UNSUPPORTED;
  if (n_requests == 0)
    return GKV_OK;
  const int64_t rows = (int64_t)n_requests * n_beams;
  const int parts = beam_parts(rows, vocab);
  const BeamWorkspace w = beam_workspace(rows, n_out);
  if (!workspace || workspace_bytes < w.total)
    return GKV_ERR_WORKSPACE;
  char *ws = (char *)workspace;
  BeamArgs a{};
  a.x = logits;
  a.stride = row_stride;
  a.cum = cum_scores;
  a.done = done;
  a.R = n_requests;
  a.K = n_beams;
  a.V = vocab;
  a.n = n_out;
  a.eos = eos;
  a.parts = parts;
  a.ml = (float2 *)ws;
  a.best = (float *)(ws + w.best);
  a.token = (int32_t *)(ws + w.token);
  a.scores = scores;
  a.parents = parents;
  a.tokens = tokens;
  a.done_out = done_out;
  a.dev_err = dev_err;
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)(rows * parts));
  if (bf)
    hipLaunchKernelGGL((beam_rows_kernel<true>), grid, dim3(kBeamThreads), 0, s, a);
  else
    hipLaunchKernelGGL((beam_rows_kernel<false>), grid, dim3(kBeamThreads), 0, s, a);
  const int st = launch_status("beam_rows_kernel");
  if (st)
    return st;
  hipLaunchKernelGGL(beam_merge_kernel, dim3((unsigned)n_requests), dim3(64 * kMergeWaves), 0, s, a);
  return launch_status("beam_merge_kernel");
}
