// Beam search's choice: for every request the n best of its beams' continuations.
//
// A continuation of beam b by token t scores cum[b] + x[b][t] - log sum_v exp x[b][v]. The
// logits are read once: a wave takes a run of a row, keeps its sum per lane, and its n best so
// far in one register across its lanes, sorted. Inside a row the order is that of the logits, so
// nothing but their values is compared until the rows meet; scores are formed and compared in 64 bits (two beams' scores differ by as little as
// their sums' last bits).
//
// A row's sum does not depend on where the row lies or how it is cut, which would decide between
// equal beams: tiles are counted from token 0, whatever the row's alignment; a lane's 16 logits
// of a tile are summed in fp32 against their largest, r, so that the sum s depends on those 16 alone;
// and s exp(r), a number of its own for the same reason, is added up in 64 bits, as a power of two
// times an fp32 number: n = rint(r log2 e), 2^n (s 2^(r log2 e - n)), log2 e in two pieces. What the
// order of the additions changes is 2^-53 of it; the fp32 sums are off by 2^-19 of theirs at most. That
// reaches over |r| <= 700; a row whose largest logit is past 600 takes a second sum, in fp32 against a
// running maximum (of masked values alone it is their number). Both together are some 20
// instructions for 16 logits: 24 x 5 rows of 200000 in bf16 25.5 us for 24.6 with the second
// alone, 64 x 8 of 131072 fp32 55.7 for 54.8.
//
// Many long rows are bound by HBM: 64 x 8 rows of 131072 fp32 logits (a tenth of them of beams that
// have ended, 242 MB), 16 best, 50 us, 4.8 TB/s, and 6 for the second launch. Where a wave has
// but a few tiles, the sorts and the first threshold show: 24 x 5 rows of 200000 in bf16, 10 best,
// 38 MB, 19.5 and 7 us; 4 rows of 32001 6.8 and 6, all of it latency.
#include "lds_dma.hpp"

#include <algorithm>

namespace gkv {

constexpr int kBeamMost = 64;      // candidates per request, at most: one a lane
constexpr int kBeamThreads = 256;  // four waves of a row's part
constexpr int kBeamWaves = kBeamThreads / 64;
constexpr int kMergeWaves = 8;
constexpr float kFloatMax = 3.402823466e38f;

// What a run of a row adds up to: the largest logit m, sum of exp(x - m), and sum of exp(x).
struct RowSum {
  float m, l;
  double sum;
};
constexpr float kPlainMost = 600.0f; // |m| up to here: sum is the one that counts

struct BeamArgs {
  const void *x;
  int64_t stride;
  const float *cum;
  const int32_t *done;
  int R, K, V, n, eos;
  int parts;        // workgroups per row
  RowSum *sums;     // [rows][parts]
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

__device__ __forceinline__ float lane_of(float x, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane));
}

// A logit and its token as one number that grows with the logit and, at equal ones, falls
// with the token (-0 as 0). 0: none.
__device__ __forceinline__ uint64_t key_of(float x, int token) {
  return (uint64_t)order_of(x + 0.0f) << 32 | (uint32_t)~token;
}
__device__ __forceinline__ float value_of(uint32_t u) { // of order_of's number
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ float logit_of(uint64_t key) { return value_of((uint32_t)(key >> 32)); }
__device__ __forceinline__ int token_of(uint64_t key) { return (int)~(uint32_t)key; }

// Between a wave's writes to LDS and its other lanes' reads: they keep their order by themselves,
// the compiler has to as well.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// The words of lane and of lane ^ X, in either order, by vector moves (an LDS swizzle's latency would
// be most of a step's).
template <int X>
__device__ __forceinline__ void pair_of(uint32_t x, uint32_t &a, uint32_t &b) {
  if (X >= 16) { // (swaps odd rows of one register with even rows of the other, or halves)
    const auto r = X == 16 ? __builtin_amdgcn_permlane16_swap(x, x, false, false)
                           : __builtin_amdgcn_permlane32_swap(x, x, false, false);
    a = r[0];
    b = r[1];
    return;
  }
  constexpr int kSwap1 = 0xb1, kSwap2 = 0x4e, kSwap3 = 0x1b, kHalfMirror = 0x141, kTurn8 = 0x128;
  constexpr int ctrl = X == 1 ? kSwap1 : X == 2 ? kSwap2 : X == 4 ? kHalfMirror : kTurn8;
  uint32_t o = __builtin_amdgcn_mov_dpp(x, ctrl, 0xf, 0xf, true);
  if (X == 4) // (lane ^ 7, then ^ 3)
    o = __builtin_amdgcn_mov_dpp(o, kSwap3, 0xf, 0xf, true);
  a = x;
  b = o;
}

// One step of a sort over the lanes: lane and lane ^ X, the larger key to the lower lane where
// down, else to the upper.
template <int X>
__device__ __forceinline__ void sort_step(uint64_t &key, bool down) {
  uint32_t a[2], b[2];
  pair_of<X>((uint32_t)key, a[0], b[0]);
  pair_of<X>((uint32_t)(key >> 32), a[1], b[1]);
  const uint64_t x = (uint64_t)a[1] << 32 | a[0], y = (uint64_t)b[1] << 32 | b[0];
  const bool lower = (threadIdx.x & X) == 0;
  key = (x > y) == (lower == down) ? x : y;
}

template <int X>
__device__ __forceinline__ void sort_step(uint32_t &key, bool down) {
  uint32_t x, y;
  pair_of<X>(key, x, y);
  const bool lower = (threadIdx.x & X) == 0;
  key = lower == down ? max(x, y) : min(x, y);
}

// Largest first, of keys that rise and then fall (or the reverse).
__device__ __forceinline__ void sort_bitonic(uint64_t &key) {
  sort_step<32>(key, true);
  sort_step<16>(key, true);
  sort_step<8>(key, true);
  sort_step<4>(key, true);
  sort_step<2>(key, true);
  sort_step<1>(key, true);
}

// The 64 lanes' keys, smallest first (so that the lanes of another, sorted the other way round, can
// be compared one by one).
template <typename Key>
__device__ __forceinline__ void sort_up(Key &key) {
  const int lane = threadIdx.x & 63;
  auto down = [&](int size) { return (lane & size) != 0; };
  sort_step<1>(key, down(2));
  sort_step<2>(key, down(4));
  sort_step<1>(key, down(4));
  sort_step<4>(key, down(8));
  sort_step<2>(key, down(8));
  sort_step<1>(key, down(8));
  sort_step<8>(key, down(16));
  sort_step<4>(key, down(16));
  sort_step<2>(key, down(16));
  sort_step<1>(key, down(16));
  sort_step<16>(key, down(32));
  sort_step<8>(key, down(32));
  sort_step<4>(key, down(32));
  sort_step<2>(key, down(32));
  sort_step<1>(key, down(32));
  sort_step<32>(key, false);
  sort_step<16>(key, false);
  sort_step<8>(key, false);
  sort_step<4>(key, false);
  sort_step<2>(key, false);
  sort_step<1>(key, false);
}

// A lane's 16 logits of tile t of a row as fp32: granules of 16 bytes, 64 lanes side by side, from
// token 0 on at whatever address the row begins (rows that begin on no 16-byte line cost little: 64 x 8
// of 131071 fp32 54.2 us, of 131072 55.7; 24 x 5 of 200001 in bf16 26.3, of 200000 25.5). Elements past
// the row are -inf and not read.
typedef uint32_t Granule __attribute__((ext_vector_type(4), aligned(2)));
template <bool BF>
struct Tile {
  static constexpr int N = BF ? 8 : 4, U = 16 / N; // of a granule; granules
  u32x4 raw[U];
  // The token that the lane's granule u begins with.
  __device__ __forceinline__ static int first(int t, int u) {
    return (t * 64 * U + u * 64 + (int)(threadIdx.x & 63)) * N;
  }
  __device__ __forceinline__ void load(const char *row, int t, int V) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int e = first(t, u);
      if (e <= V - N) {
        raw[u] = __builtin_nontemporal_load((const Granule *)(row + (int64_t)e * (BF ? 2 : 4)));
      } else {
        float v[N];
#pragma unroll
        for (int j = 0; j < N; j++) {
          v[j] = -INFINITY;
          if (e + j < V)
            v[j] = BF ? bf16_to_f32(((const uint16_t *)row)[e + j]) : ((const float *)row)[e + j];
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
          raw[u][j] = BF ? __float_as_uint(v[2 * j % N]) >> 16 | __float_as_uint(v[(2 * j + 1) % N])
                         : __float_as_uint(v[j % N]);
      }
    }
  }
  __device__ __forceinline__ float at(int k) const { // element k of the lane's 16
    if (BF)
      return __uint_as_float(k & 1 ? raw[k / 8][k % 8 / 2] & 0xffff0000u : raw[k / 8][k % 8 / 2] << 16);
    return __uint_as_float(raw[k / 4 % U][k % 4]);
  }
};

// What the waves of a workgroup tell each other, in LDS: their n-th best so far, and what their first
// tiles said of the four together. (Typed as LDS: a volatile access through a plain pointer would be one
// to memory of any kind, which waits for the tiles under way.)
typedef volatile __attribute__((address_space(3))) float *Told;
constexpr int kListMost = 63 + 16 * 64; // candidates of a wave: fewer than a sort's, and a tile

// One wave's tiles t0 .. t1 - 1 of a row: sums per lane, and the 64 best keys, best in lane 0.
// What may be among the row's n best is put into the wave's list in LDS, 64 at a time are
// sorted and joined with the best so far: a few hundred instructions for 64 candidates, where
// putting them in one by one took some 80 each. Where it meets a NaN or +inf, at.l ends as NaN, and
// the caller runs it again with PLAIN, which looks at every value.
// low: the waves' n-th best so far: what is below one of them is not among the row's n
// best, whoever reads it when. The waves begin with what their first tiles say: the n-th largest
// of one wave's lanes' maxima, or the least of the four waves' n / 4-th.
template <bool BF, bool PLAIN>
__device__ __forceinline__ void row_part(const BeamArgs &a, const char *row, int t0, int t1, Told low,
                                         uint64_t *list, uint64_t &best, RowSum &at) {
  constexpr int N = Tile<BF>::N;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  best = 0;
  float m = -kFloatMax, l = 0.0f;
  double sum = 0;
  float over = -INFINITY; // the least logit that may join: above the n-th best, whose token is lower
  int listed = 0;
  auto join = [&]() { // the last 64 of the list with the best
    wave_sync();
    listed = max(listed - 64, 0);
    uint64_t key = list[listed + lane];
    sort_up(key);
    best = best > key ? best : key;
    sort_bitonic(best);
    const uint32_t nth = __builtin_amdgcn_readlane((uint32_t)(best >> 32), a.n - 1); // (0: there are fewer)
    wave_sync();
    if (nth != 0) {
      over = value_of(nth + 1);
      if (lane == 0 && value_of(nth) > low[wave])
        low[wave] = value_of(nth);
    }
  };
  Tile<BF> tile[2]; // one looked at, one under way (two: 50.5 us for 49.3, 64 x 8 rows of 131072)
#pragma unroll
  for (int i = 0; i < 2; i++)
    if (t0 + i < t1)
      tile[i].load(row, t0 + i, a.V);
  {
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 2; i++)
      if (t0 + i < t1)
#pragma unroll
        for (int k = 0; k < 16; k++)
          mx = fmaxf(mx, PLAIN ? plain_logit(tile[i].at(k)) : tile[i].at(k));
    uint32_t top = order_of(mx);
    sort_up(top);
    mx = value_of(top);
    if (lane == 64 - a.n)
      low[wave] = mx;
    if (lane == 64 - (a.n + kBeamWaves - 1) / kBeamWaves)
      low[kBeamWaves + wave] = mx;
    lds_barrier();
  }
  const float fourth = fminf(fminf(low[4], low[5]), fminf(low[6], low[7]));
  auto look = [&](Tile<BF> &now, int t) {
    float x[16], top[4], mx; // the largest of four, of all
    const float l0 = low[0], l1 = low[1], l2 = low[2], l3 = low[3]; // (here: nothing waits for them yet)
#pragma unroll
    for (int k = 0; k < 16; k++)
      x[k] = PLAIN ? plain_logit(now.at(k)) : now.at(k);
#pragma unroll
    for (int q = 0; q < 4; q++)
      top[q] = fmaxf(fmaxf(x[4 * q], x[4 * q + 1]), fmaxf(x[4 * q + 2], x[4 * q + 3]));
    mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
    const float r = fmaxf(mx, -kFloatMax);
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < 16; k++)
      s += __builtin_amdgcn_exp2f((x[k] - r) * kLog2e);
    {
      constexpr float kLog2eRest = 1.925963033e-8f; // log2 e - kLog2e
      const float y = fminf(fmaxf(r, -1000.0f), 1000.0f); // (past 700 the power of two is 0 or inf)
      const float n = __builtin_rintf(y * kLog2e);
      const float p = __builtin_amdgcn_exp2f(fmaf(y, kLog2eRest, fmaf(y, kLog2e, -n)));
      sum += __builtin_ldexp((double)(s * p), (int)n);
      const float f = __builtin_amdgcn_exp2f(-fabsf(m - r) * kLog2e);
      l = r > m ? fmaf(l, f, s) : fmaf(s, f, l);
      m = fmaxf(m, r);
    }
    const float least = fmaxf(fmaxf(fmaxf(l0, l1), fmaxf(l2, l3)), fmaxf(fourth, over));
    if (__any(mx >= least)) {
#pragma unroll
      for (int q = 0; q < 4; q++) {
        if (!__any(top[q] >= least))
          continue;
#pragma unroll
        for (int k = 4 * q; k < 4 * q + 4; k++) {
          if (!__any(x[k] >= least))
            continue;
          const int e = Tile<BF>::first(t, k / N) + k % N;
          const bool in = e < a.V && x[k] >= least;
          const uint64_t who = __ballot(in);
          if (in)
            list[listed + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32),
                                                    __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0))] =
                key_of(x[k], e);
          listed += __popcll(who);
        }
      }
    }
    if (t + 2 < t1)
      now.load(row, t + 2, a.V);
    while (listed >= 64)
      join();
  };
  for (int t = t0; t < t1; t += 2) {
    look(tile[0], t);
    if (t + 1 < t1)
      look(tile[1], t + 1);
  }
  if (listed > 0) {
    if (lane >= listed) // (what the sort takes beside them: none)
      list[lane] = 0;
    join();
  }
  at = RowSum{m, l, sum};
}

template <bool BF>
__global__ __launch_bounds__(kBeamThreads) void beam_rows_kernel(BeamArgs a) {
  __shared__ uint64_t s_list[kBeamWaves][kListMost]; // candidates; then every wave's best
  __shared__ RowSum s_sums[kBeamWaves];
  __shared__ float s_low[2][2 * kBeamWaves];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int row = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  // (a row that is finished, or that no score can reach, is not read)
  const float cum = a.cum[row];
  if ((a.done && a.done[row] != 0) || !(cum > -INFINITY))
    return;
  const char *start = (const char *)a.x + (int64_t)row * a.stride * (BF ? 2 : 4);
  // this wave's tiles, in order
  const int tiles = (int)(((int64_t)a.V + 1023) / 1024);
  const int64_t w = (int64_t)part * kBeamWaves + wave, n_waves = (int64_t)a.parts * kBeamWaves;
  const int t0 = (int)(w * tiles / n_waves), t1 = (int)((w + 1) * tiles / n_waves);
  uint64_t best;
  RowSum at;
  row_part<BF, false>(a, start, t0, t1, (Told)s_low[0], s_list[wave], best, at);
  if (__syncthreads_or(at.l != at.l)) {
    // (all waves again: what bounded them may have been taken from a NaN)
    if (threadIdx.x == 0 && a.dev_err)
      atomicOr(a.dev_err, GKV_DEVERR_RANGE);
    row_part<BF, true>(a, start, t0, t1, (Told)s_low[1], s_list[wave], best, at);
  }
  // the lanes' sums, then the waves'
  auto join = [&](const RowSum &x) {
    const float mn = fmaxf(at.m, x.m);
    at.l = at.l * __builtin_amdgcn_exp2f((at.m - mn) * kLog2e) +
           x.l * __builtin_amdgcn_exp2f((x.m - mn) * kLog2e);
    at.m = mn;
    at.sum += x.sum;
  };
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1)
    join(RowSum{__shfl_xor(at.m, o), __shfl_xor(at.l, o), __shfl_xor(at.sum, o)});
  if (lane == 0)
    s_sums[wave] = at;
  s_list[wave][lane] = best;
  __syncthreads();
  const int64_t piece = (int64_t)row * a.parts + part;
  if (threadIdx.x == 0) {
    for (int k = 1; k < kBeamWaves; k++)
      join(s_sums[k]);
    a.sums[piece] = at;
  }
  // the first wave: the waves' best to the n best of all
  if (wave != 0)
    return;
#pragma unroll
  for (int k = 1; k < kBeamWaves; k++) {
    const uint64_t key = s_list[k][63 - lane];
    best = best > key ? best : key;
    sort_bitonic(best);
  }
  if (lane < a.n) {
    a.best[piece * a.n + lane] = logit_of(best);
    a.token[piece * a.n + lane] = best != 0 ? token_of(best) : -1;
  }
}

// A workgroup per request. First one or more waves per row: the parts' sums to the row's, the
// parts' best, sorted as they are, joined one by one to its n best, and their scores. Then
// an entry's place among all: in each other row, which is sorted, those before it are found by
// halving; as many threads an entry as there are, each for some of the rows.
__global__ __launch_bounds__(64 * kMergeWaves) void beam_merge_kernel(BeamArgs a) {
  extern __shared__ double s_score[];               // [K n] scores, then their tokens
  int *s_token = (int *)(s_score + a.K * a.n);      // (-1: none)
  __shared__ uint64_t s_best[kMergeWaves][64];
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  int shares = 1; // waves per row
  while (2 * shares * a.K <= kMergeWaves && 2 * shares <= a.parts)
    shares *= 2;
  for (int k0 = 0; k0 < a.K; k0 += kMergeWaves / shares) {
    const int k = k0 + wave / shares, share = wave % shares, row = r * a.K + min(k, a.K - 1);
    const float cum = a.cum[row];
    const double c = cum != cum ? -INFINITY : (double)fminf(cum, kFloatMax);
    const bool done = a.done && a.done[row] != 0;
    const bool reads = k < a.K && !done && c > -INFINITY;
    uint64_t best = 0;
    if (reads) {
      const float *xs = a.best + (int64_t)row * a.parts * a.n;
      const int32_t *ts = a.token + (int64_t)row * a.parts * a.n;
      const int e = min(63 - lane, a.n - 1); // (the other way round, so that a maximum joins them)
      constexpr int A = 4; // loads under way
      for (int p0 = share; p0 < a.parts; p0 += A * shares) {
        float x[A];
        int t[A];
#pragma unroll
        for (int i = 0; i < A; i++) {
          const int p = min(p0 + i * shares, a.parts - 1);
          x[i] = xs[p * a.n + e];
          t[i] = ts[p * a.n + e];
        }
#pragma unroll
        for (int i = 0; i < A; i++)
          if (p0 + i * shares < a.parts) {
            const uint64_t key = 63 - lane < a.n && t[i] >= 0 ? key_of(x[i], t[i]) : 0;
            best = best > key ? best : key;
            sort_bitonic(best);
          }
      }
    }
    if (shares > 1) { // (then all rows are taken at once)
      s_best[wave][lane] = best;
      __syncthreads();
    }
    if (k >= a.K || share != 0)
      continue;
    if (!(cum <= kFloatMax) && lane == 0 && a.dev_err)
      atomicOr(a.dev_err, GKV_DEVERR_RANGE);
    if (!reads) { // its one continuation, and tokens that score -inf
      if (lane < a.n) {
        s_score[k * a.n + lane] = done && lane == 0 ? c : -INFINITY;
        s_token[k * a.n + lane] = !done ? lane : lane == 0 ? a.eos : lane - 1 < a.eos ? lane - 1 : lane;
      }
      continue;
    }
    for (int i = 1; i < shares; i++) {
      const uint64_t key = s_best[wave + i][63 - lane];
      best = best > key ? best : key;
      sort_bitonic(best);
    }
    const RowSum *sums = a.sums + (int64_t)row * a.parts;
    float m = -kFloatMax;
    for (int p = lane; p < a.parts; p += 64)
      m = fmaxf(m, sums[p].m);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1)
      m = fmaxf(m, __shfl_xor(m, o));
    const bool plain = fabsf(m) <= kPlainMost;
    double l = 0;
    for (int p = lane; p < a.parts; p += 64)
      l += plain ? sums[p].sum : (double)sums[p].l * exp2(((double)sums[p].m - (double)m) * 1.4426950408889634);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1)
      l += __shfl_xor(l, o);
    // (a row of -inf alone: every score is -inf)
    const double lse = plain ? log(l) : l > 0 ? (double)m + log(l) : 0.0;
    if (lane < a.n) {
      s_score[k * a.n + lane] = c + ((double)logit_of(best) - lse);
      s_token[k * a.n + lane] = token_of(best);
    }
  }
  __syncthreads();
  // every row has n: n <= V
  const int all = a.K * a.n;
  int each = 1; // threads an entry
  while (each < 64 && 2 * each * all <= 64 * kMergeWaves)
    each *= 2;
  for (int e0 = 0; e0 < all; e0 += 64 * kMergeWaves / each) {
    const int e = e0 + tid / each, k = min(e, all - 1) / a.n;
    const double s = s_score[min(e, all - 1)];
    const int t = s_token[min(e, all - 1)];
    int place = 0;
    for (int o = tid % each; o < a.K; o += each) {
      int lo = 0, hi = o == k ? 0 : a.n; // of equal scores the lower row's come first
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        const double x = s_score[o * a.n + mid];
        if (x > s || (x == s && o < k))
          lo = mid + 1;
        else
          hi = mid;
      }
      place += o == k ? e - k * a.n : lo;
    }
    for (int o = 1; o < each; o *= 2)
      place += __shfl_xor(place, o);
    if (e < all && tid % each == 0 && place < a.n) {
      const int64_t o = (int64_t)r * a.n + place;
      const int row = r * a.K + k;
      a.scores[o] = (float)s;
      a.parents[o] = row;
      a.tokens[o] = t;
      if (a.done_out)
        a.done_out[o] = t == a.eos || (a.done && a.done[row] != 0);
    }
  }
}

// Workgroups per row: as many as give every CU sixteen waves, as long as a wave keeps a tile of
// 1024 logits (24 x 5 rows of 200000 in bf16, both launches: 512 workgroups 28 us, 1024 27, 2048
// 31; 64 x 8 of 131072 level).
constexpr int kBeamWgs = 1024;
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
  w.best = up(pieces * sizeof(RowSum));
  w.token = w.best + up(pieces * n * 4);
  w.total = w.token + pieces * n * 4;
  return w;
}

static bool beam_sizes_ok(int32_t R, int32_t K, int32_t V, int32_t n) {
  return R >= 0 && K > 0 && V > 0 && V <= 1 << 30 && n > 0 && n <= V && n <= kBeamMost && K <= kBeamMost &&
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
  a.sums = (RowSum *)ws;
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
  hipLaunchKernelGGL(beam_merge_kernel, dim3((unsigned)n_requests), dim3(64 * kMergeWaves),
                     (size_t)n_beams * n_out * 12, s, a);
  return launch_status("beam_merge_kernel");
}
