// Decode attention over a cache of whole blocks: bf16, or e4m3 codes with one
// scale per block and kv head; every position, or a sliding window and the first
// tokens that stay visible.
//
// One query token per sequence and head: score = q.k / 8, softmax over the
// positions seen and (if given) the head's sink logit, out = sum p v. Each K and V
// byte is read once for the whole group of query heads; 2 * 64 * 2 operations a
// head and token against 128 (bf16: 256) bytes a kv head and token: bound by HBM.
//
// Matrix cores, 16x16 output, K = 32, the operand arrangement of the block
// layouts (kv_append.hpp): S^T = K Q^T and O^T += V^T P^T, columns 0..7 the high
// pieces of query head col's q and p, columns 8..15 the rest, added afterwards.
// Block codes enter without their scale, which is one number per block and
// wave: K's goes into the factor of the exponent, V's into the weights, so the
// stream costs no scale loads per token. Against codes q is split into fp16 pieces
// (e4m3 values are fp16 values; 22 bits of q, scaled by a power of two per head so
// that no range is lost), against bf16 K into bf16 pieces (16 bits); p always into
// bf16 pieces (its range is that of exp2). Two bf16 pieces leave up to 2^-18 of a
// value, 2^-9 of a bf16 output's own rounding; an fp32 output takes three, the
// third through matrix ops of its own (FINE).
//
// A step is two blocks (32 tokens). A wave takes the steps of one (sequence, kv
// head), loads the next step's blocks while it computes this one's, and leaves it
// to the other waves of its SIMD to cover the chain of matrix op, exponential,
// matrix op: 2 steps in registers, 4 waves per SIMD, with ranges 2 (3 or 4 steps
// and 3 or 5 waves measured the same or worse). Two ways to deal the steps out:
//   whole   contexts and windows that are not long: a (sequence, kv head) belongs
//           to 1 .. 8 waves of one workgroup, which cut its steps and merge in LDS.
//           One launch, no workspace. 512 sequences of 129 .. 2049 tokens (8 kv
//           heads, codes, 586 MB): 107 us, 5.5 TB/s; 97 windows of 4096 behind 64
//           (411 MB): 70 us, 5.9 TB/s.
//   ranges  the sequences laid end to end are cut into equal ranges, one per
//           wave; every workgroup finds its own range from the lengths
//           in its prologue. A sequence inside one range is finished there,
//           the pieces of the others go to the workspace and a second launch
//           merges them, a workgroup per range. 4 sequences of 129 .. 16384 tokens:
//           18 us, where one workgroup a sequence and head takes 43.
#include "kept_attend.hpp"

#include <algorithm>

namespace gkv {

// Range workgroups: one per CU, two waves a SIMD. Two per CU make twice the pieces
// and shorter ranges (us, 256 / 512 workgroups: 32 sequences of 129 .. 16384
// tokens 55.7 / 60.4, bf16 100 / 108; 4 of them 18.4 / 20.6, 22.1 / 28.3).
constexpr int kSplitWgs = 256;
constexpr int kMinRangeSteps = 4;      // steps per range, at least
constexpr int kMergeThreads = 512;
constexpr int kMaxRanges = 8 * kSplitWgs; // one kv head: 8 ranges a workgroup

// ---- whole: one workgroup holds every step of its (sequence, kv head)s --------------

template <bool BLK, int R, int WPE, bool FINE>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(WPE)))
void kept_decode_whole_kernel(KeptDecodeArgs a) {
  __shared__ float s_o[8][kPieceFloats];
  __shared__ float2 s_ml[8][kHeads];
  const int n_groups = (a.n_kv_heads + a.heads_per_wg - 1) / a.heads_per_wg;
  const int b = blockIdx.x / n_groups;
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int slot = wave / a.parts, part = wave % a.parts;
  const int g = (int)(blockIdx.x % n_groups) * a.heads_per_wg + slot;
  const int len = uniform(a.seq_lens[b]);
  if (len > a.max_len && threadIdx.x == 0 && a.dev_err)
    atomicOr(a.dev_err, GKV_DEVERR_LENGTH);
  const Span sp = span_of(a, max(min(len, a.max_len), 0));
  const int n = span_steps(sp);
  const bool ok = g < a.n_kv_heads;
  if (n == 0) { // an empty sequence: zeros
    if (ok)
      put_zeros(a, (int64_t)b * a.out_stride + (int64_t)g * a.G * kHeadDim, a.G * kHeadDim,
                part * 64 + lane, a.parts * 64);
    return;
  }
  State st;
  if (ok) {
    const int s0 = part * n / a.parts, s1 = (part + 1) * n / a.parts;
    if (s0 < s1) {
      st = attend<BLK, R, FINE>(a, b, g, sp, s0, s1);
    } else {
      st.m = kLowest;
      st.l = 0.0f;
#pragma unroll
      for (int nn = 0; nn < 4; nn++)
        st.o[nn] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    if (a.parts == 1) {
      put_whole(a, b, g, st);
      return;
    }
    const int col = lane & 15, kg = lane >> 4;
    if (col < kHeads) {
#pragma unroll
      for (int nn = 0; nn < 4; nn++)
        *(f32x4 *)&s_o[wave][col * kHeadDim + 16 * nn + 4 * kg] = st.o[nn];
      if (kg == 0)
        s_ml[wave][col] = float2{st.m, st.l};
    }
  }
  if (a.parts == 1)
    return;
  __syncthreads();
  if (!ok)
    return;
  // the parts' sums against their common maximum, 4 dims a thread
  const int w0 = slot * a.parts;
  for (int e = part * 64 + lane; e < a.G * (kHeadDim / 4); e += a.parts * 64) {
    const int h = e / (kHeadDim / 4);
    float m = kLowest, l = 0.0f;
    for (int p = 0; p < a.parts; p++)
      m = fmaxf(m, s_ml[w0 + p][h].x);
    f32x4 o{0.0f, 0.0f, 0.0f, 0.0f};
    for (int p = 0; p < a.parts; p++) {
      const float f = __builtin_amdgcn_exp2f(s_ml[w0 + p][h].x - m);
      l = fmaf(s_ml[w0 + p][h].y, f, l);
      o += *(const f32x4 *)&s_o[w0 + p][4 * e] * f;
    }
    put(a.out, (int64_t)b * a.out_stride + (int64_t)g * a.G * kHeadDim + 4 * e,
        o * out_factor(m, l, sink_of(a, g, h)), a.out_bf16);
  }
}

// ---- ranges ----------------------------------------------------------------------
//
// (About 30 scalar registers of the prologue and the loop over sequences wait in lanes of a
// vector register while a wave is in its steps; nothing goes to memory.)

// Range r of the T steps cut into n (n <= 2048): floor(r T / n), in 32 bits.
__device__ __forceinline__ int range_begin(int r, int T, int n) {
  const uint32_t q = (uint32_t)T / (uint32_t)n, m = (uint32_t)T % (uint32_t)n;
  return (int)(r * q + r * m / (uint32_t)n);
}

// The range that holds step p.
__device__ __forceinline__ int range_of(int p, int T, int n) {
  return (int)(((int64_t)(p + 1) * n - 1) / T);
}

template <bool BLK, int R, int WPE, bool FINE>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(WPE)))
void kept_decode_split_kernel(KeptDecodeArgs a) {
  __shared__ int s_wave[8];
  __shared__ int s_b[8], s_c[8];
  const int t = threadIdx.x, lane = t & 63, wave = uniform(t >> 6), nt = blockDim.x;
  const int n_waves = nt >> 6, subs = n_waves / a.n_kv_heads; // ranges in this workgroup

  // Prefix sums of the sequences' steps: thread t holds sequences t * per ..
  const int per = (a.B + nt - 1) / nt;
  const int b0 = min(t * per, a.B), b1 = min(b0 + per, a.B);
  int mine = 0;
  bool over = false;
  for (int b = b0; b < b1; b++) {
    over |= a.seq_lens[b] > a.max_len;
    mine += span_steps(span_of(a, span_len(a, b)));
  }
  int incl = mine;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int v = __shfl_up(incl, off, 64);
    if (lane >= off)
      incl += v;
  }
  if (lane == 63)
    s_wave[wave] = incl;
  __syncthreads();
  int before = 0, T = 0;
  for (int w = 0; w < n_waves; w++) {
    const int v = s_wave[w];
    before += w < wave ? v : 0;
    T += v;
  }
  T = uniform(T);
  const int n = min(a.max_ranges, max(T / kMinRangeSteps, 1));
  const int r0 = blockIdx.x * subs;
  int c = before + incl - mine;
  // each of the workgroup's ranges: the sequence that holds its first step
  int at[8];
#pragma unroll
  for (int k = 0; k < 8; k++)
    at[k] = k < subs && r0 + k < n ? range_begin(r0 + k, T, n) : -1;
  for (int b = b0; b < b1; b++) {
    const int m = span_steps(span_of(a, span_len(a, b)));
#pragma unroll
    for (int k = 0; k < 8; k++)
      if (c <= at[k] && at[k] < c + m) {
        s_b[k] = b;
        s_c[k] = c;
        a.cuts[r0 + k] = int4{c < at[k] ? b : -1, c, c + m, T};
      }
    c += m;
  }
  if (t < subs && (r0 + t >= n || T == 0))
    a.cuts[r0 + t] = int4{-1, 0, 0, 0};
  if (blockIdx.x == 0 && over && a.dev_err)
    atomicOr(a.dev_err, GKV_DEVERR_LENGTH);
  // sequences without tokens: zeros
  for (int b = blockIdx.x; b < a.B; b += gridDim.x)
    if (a.seq_lens[b] <= 0 || a.max_len <= 0)
      put_zeros(a, (int64_t)b * a.out_stride, a.n_kv_heads * a.G * kHeadDim, t, nt);
  __syncthreads();

  const int sub = wave / a.n_kv_heads, g = wave % a.n_kv_heads;
  const int r = r0 + sub;
  if (r >= n || T == 0)
    return;
  const int rs = range_begin(r, T, n), re = range_begin(r + 1, T, n);
  int b = uniform(s_b[sub]), cb = uniform(s_c[sub]);
  while (cb < re) {
    const Span sp = span_of(a, uniform(span_len(a, b)));
    const int m = span_steps(sp);
    const int s0 = max(rs - cb, 0), s1 = min(re - cb, m);
    if (s0 < s1) {
      const State st = attend<BLK, R, FINE>(a, b, g, sp, s0, s1);
      if (s0 == 0 && s1 == m) {
        put_whole(a, b, g, st);
      } else {
        const int col = lane & 15, kg = lane >> 4;
        const int64_t piece = ((int64_t)r * 2 + (cb + s0 == rs ? 0 : 1)) * a.n_kv_heads + g;
        if (col < kHeads) {
          float *o = a.ws_o + piece * kPieceFloats + col * kHeadDim + 4 * kg;
#pragma unroll
          for (int nn = 0; nn < 4; nn++)
            *(f32x4 *)(o + 16 * nn) = st.o[nn];
          if (kg == 0)
            *(float2 *)(a.ws_ml + piece * kPieceMl + 2 * col) = float2{st.m, st.l};
        }
      }
    }
    cb += m;
    b++;
  }
}

// The pieces of a sequence that was cut: M = max m_i, out = sum o_i 2^(m_i - M) /
// (sum l_i 2^(m_i - M) + 2^(sink - M)). One workgroup per range, whose record
// (left by the split) names the sequence that the range starts inside of. A
// sequence of at most kMergeFew pieces is merged by the first such range's, a
// wave per kv head, every piece's loads at once. The kv heads of a longer one are
// dealt over all of them, a wave taking every eighth piece, four at a time, the waves
// joined in LDS. In one of more pieces than there are query heads each of those
// has a workgroup: 16 threads a piece (4 dims each), 32 pieces at a time, the first
// four of each thread loaded before the weights are known. Bound by latency: the
// record, then the pieces.
constexpr int kMergeFew = 4;
__global__ __launch_bounds__(kMergeThreads) void kept_decode_merge_kernel(KeptDecodeArgs a) {
  constexpr int D = kHeadDim, kWaves = kMergeThreads / 64, kGroups = kMergeThreads / 16;
  __shared__ float s_w[kMaxRanges];
  __shared__ float s_red[kWaves];
  __shared__ f32x4 s_o[kWaves][64][2];
  __shared__ float2 s_ml[kWaves][kHeads];
  const int4 cut = a.cuts[blockIdx.x];
  if (cut.x < 0)
    return;
  const int T = cut.w, n = min(a.max_ranges, max(T / kMinRangeSteps, 1)), b = cut.x;
  const int w0 = range_of(cut.y, T, n), np = range_of(cut.z - 1, T, n) - w0 + 1;
  const int inside = (int)blockIdx.x - w0 - 1;
  if (np <= kMergeFew && inside > 0)
    return;
  // the first piece is its range's last one, unless the sequence starts there
  const int first_slot = range_begin(w0, T, n) < cut.y ? 1 : 0;
  auto piece = [&](int i, int g) {
    return ((int64_t)(w0 + i) * 2 + (i == 0 ? first_slot : 0)) * a.n_kv_heads + g;
  };
  const int t = threadIdx.x, lane = t & 63, wave = uniform(t >> 6);
  if (np <= kMergeFew) {
    const int g = wave, h = lane >> 3, d0 = 8 * (lane & 7);
    if (g >= a.n_kv_heads || h >= a.G)
      return;
    float2 ml[kMergeFew];
    f32x4 x[kMergeFew][2];
#pragma unroll
    for (int i = 0; i < kMergeFew; i++) {
      const int64_t p = piece(min(i, np - 1), g);
      ml[i] = *(const float2 *)(a.ws_ml + p * kPieceMl + 2 * h);
      const f32x4 *o = (const f32x4 *)(a.ws_o + p * kPieceFloats + h * D + d0);
      x[i][0] = o[0];
      x[i][1] = o[1];
    }
    float m = kLowest, l = 0.0f;
#pragma unroll
    for (int i = 0; i < kMergeFew; i++)
      m = fmaxf(m, ml[i].x);
    f32x4 o0{0.0f, 0.0f, 0.0f, 0.0f}, o1{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kMergeFew; i++)
      if (i < np) {
        const float f = __builtin_amdgcn_exp2f(ml[i].x - m);
        l = fmaf(ml[i].y, f, l);
        o0 += x[i][0] * f;
        o1 += x[i][1] * f;
      }
    const float f = out_factor(m, l, sink_of(a, g, h));
    const int64_t ob = (int64_t)b * a.out_stride + (int64_t)(g * a.G + h) * D + d0;
    put(a.out, ob, o0 * f, a.out_bf16);
    put(a.out, ob + 4, o1 * f, a.out_bf16);
    return;
  }
  if (np - 1 < a.n_kv_heads * a.G) {
    const int h = lane >> 3, d0 = 8 * (lane & 7), hc = min(h, a.G - 1);
    for (int g = inside; g < a.n_kv_heads; g += np - 1) {
      float m = kLowest, l = 0.0f;
      f32x4 o0{0.0f, 0.0f, 0.0f, 0.0f}, o1{0.0f, 0.0f, 0.0f, 0.0f};
      for (int i0 = wave; i0 < np; i0 += 4 * kWaves) {
        float2 ml[4];
        f32x4 x[4][2];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int64_t p = piece(min(i0 + j * kWaves, np - 1), g);
          ml[j] = *(const float2 *)(a.ws_ml + p * kPieceMl + 2 * hc);
          const f32x4 *o = (const f32x4 *)(a.ws_o + p * kPieceFloats + hc * D + d0);
          x[j][0] = o[0];
          x[j][1] = o[1];
        }
        float mn = m;
#pragma unroll
        for (int j = 0; j < 4; j++)
          mn = fmaxf(mn, ml[j].x); // (a repeated last piece moves no maximum)
        const float f0 = __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= f0;
        o0 *= f0;
        o1 *= f0;
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (i0 + j * kWaves < np) {
            const float f = __builtin_amdgcn_exp2f(ml[j].x - m);
            l = fmaf(ml[j].y, f, l);
            o0 += x[j][0] * f;
            o1 += x[j][1] * f;
          }
      }
      __syncthreads(); // (the arrays may still be read for another head)
      s_o[wave][lane][0] = o0;
      s_o[wave][lane][1] = o1;
      if ((lane & 7) == 0)
        s_ml[wave][h] = float2{m, l};
      __syncthreads();
      // thread t < 128: 4 dims of query head t / 16
      const int th = t / 16;
      if (t < 128 && th < a.G) {
        float mt = kLowest, lt = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; w++)
          mt = fmaxf(mt, s_ml[w][th].x);
        f32x4 ot{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
          const float f = __builtin_amdgcn_exp2f(s_ml[w][th].x - mt);
          lt = fmaf(s_ml[w][th].y, f, lt);
          ot += s_o[w][t / 2][t & 1] * f;
        }
        put(a.out, (int64_t)b * a.out_stride + (int64_t)g * a.G * D + 4 * t,
            ot * out_factor(mt, lt, sink_of(a, g, th)), a.out_bf16);
      }
    }
    return;
  }
  const int grp = t >> 4, e = t & 15;
  for (int item = inside; item < a.n_kv_heads * a.G; item += np - 1) {
    const int g = item / a.G, h = item % a.G;
    auto load = [&](int i) {
      return *(const f32x4 *)(a.ws_o + piece(min(i, np - 1), g) * kPieceFloats + h * D + 4 * e);
    };
    f32x4 x[4];
#pragma unroll
    for (int j = 0; j < 4; j++)
      x[j] = load(grp + j * kGroups);
    // the common maximum, the pieces' weights, the sum
    float m = kLowest;
    for (int i = t; i < np; i += kMergeThreads)
      m = fmaxf(m, a.ws_ml[piece(i, g) * kPieceMl + 2 * h]);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1)
      m = fmaxf(m, __shfl_xor(m, off));
    __syncthreads(); // (the arrays may still be read for another head)
    if (lane == 0)
      s_red[wave] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; w++)
      m = fmaxf(m, s_red[w]);
    float l = 0.0f;
    for (int i = t; i < np; i += kMergeThreads) {
      const float2 ml = *(const float2 *)(a.ws_ml + piece(i, g) * kPieceMl + 2 * h);
      const float f = __builtin_amdgcn_exp2f(ml.x - m);
      s_w[i] = f;
      l = fmaf(ml.y, f, l);
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1)
      l += __shfl_xor(l, off);
    __syncthreads();
    if (lane == 0)
      s_red[wave] = l;
    f32x4 o{0.0f, 0.0f, 0.0f, 0.0f};
    for (int i = grp; i < np; i += 4 * kGroups) {
      f32x4 y[4];
#pragma unroll
      for (int j = 0; j < 4; j++)
        y[j] = i + 4 * kGroups < np ? load(i + (4 + j) * kGroups) : x[j];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if (i + j * kGroups < np)
          o += x[j] * s_w[i + j * kGroups];
        x[j] = y[j];
      }
    }
#pragma unroll
    for (int off = 16; off <= 32; off <<= 1)
#pragma unroll
      for (int r = 0; r < 4; r++)
        o[r] += __shfl_xor(o[r], off);
    if (lane < 16)
      s_o[wave][lane][0] = o;
    __syncthreads();
    if (t < 16) {
      o = s_o[0][t][0];
      l = s_red[0];
#pragma unroll
      for (int w = 1; w < kWaves; w++) {
        o += s_o[w][t][0];
        l += s_red[w];
      }
      put(a.out, (int64_t)b * a.out_stride + (int64_t)(g * a.G + h) * D + 4 * t,
          o * out_factor(m, l, sink_of(a, g, h)), a.out_bf16);
    }
  }
}

// ---- host side --------------------------------------------------------------------

// Steps of the longest sequence that a call with these bounds can meet.
static int64_t steps_bound(int32_t max_seq_len, int32_t kept, int32_t window) {
  int64_t blocks = ((int64_t)max_seq_len + kBlockTokens - 1) / kBlockTokens;
  if (window > 0)
    blocks = std::min<int64_t>(blocks, ((int64_t)kept + window) / kBlockTokens + 1);
  return (blocks + 1) / 2;
}

// Whole sequences or ranges. A wave takes about 1 us for a step (bf16: 1.2), eight
// share a sequence, so the longest one costs steps / 8 us whatever the rest do;
// ranges cost a second launch and their pieces, 5 to 10 us, but no sequence is
// longer than the others. Measured (us, whole / ranges, 8 heads, codes): 512
// sequences of 129 .. 2049 tokens 110 / 116 (bf16 192 / 209), 16 of them 10.7 /
// 17.0; 128 of 129 .. 4096 56 / 58, 8 of them 16.0 / 16.8 (bf16 19.1 / 18.0); 8 of
// 129 .. 8192 26 / 19, 4 of 129 .. 16384 43 / 18. A window of 4096 behind 16: 97
// sequences 68 / 76, 32 of them 25 / 34, 8 of them 18 / 16 (bf16 25 / 21).
constexpr int kWholeSteps = 72;      // whole whatever the number of sequences
constexpr int kWholeStepsMany = 144; // whole for this many (sequence, head)s
constexpr int kWholeMany = 96;
static bool use_whole(int32_t B, int32_t n_kv_heads, int32_t max_seq_len, int32_t kept,
                      int32_t window) {
  const int64_t steps = steps_bound(max_seq_len, kept, window);
  return steps <= kWholeSteps ||
         (steps <= kWholeStepsMany && (int64_t)B * n_kv_heads >= kWholeMany);
}

// Waves per (sequence, head) of the whole kernel. As many as take half the GPU's
// 4096 wave slots: more leave each wave too few steps (a window of 128: 512
// sequences 19 us with one, 32 with four) without reading faster. Contexts without a window differ
// in length, so there a wave gets at most 16 steps and the last sequences end
// sooner (512 sequences of 129 .. 2049 tokens: 126 us with one wave, 114, 108,
// 110 with 2, 4, 8; bf16 226, 206, 196, 189).
constexpr int kWholeWaves = 2048;
static int whole_parts(int32_t B, int32_t n_kv_heads, int64_t steps, int32_t window) {
  int parts = 1;
  while (parts < 8 && 2 * parts <= steps &&
         (2 * parts * (int64_t)B * n_kv_heads <= kWholeWaves ||
          (window == 0 && steps > 16 * parts)))
    parts *= 2;
  return parts;
}

static int range_subs(int n_kv_heads) { return 8 / n_kv_heads; }

struct KeptWorkspace {
  size_t ml, o, total; // (the ranges' records come first)
};
static KeptWorkspace kept_workspace(int32_t n_kv_heads) {
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  const size_t pieces = (size_t)kSplitWgs * range_subs(n_kv_heads) * 2 * n_kv_heads;
  KeptWorkspace w;
  w.ml = up((size_t)kSplitWgs * range_subs(n_kv_heads) * sizeof(int4));
  w.o = w.ml + up(pieces * kPieceMl * 4);
  w.total = w.o + pieces * kPieceFloats * 4;
  return w;
}

} // namespace gkv

extern "C" size_t gkv_kept_workspace_bytes(int32_t B, int32_t n_kv_heads, int32_t max_seq_len,
                                           int32_t kept, int32_t window) {
  using namespace gkv;
  // (what the call of any smaller batch needs too)
  if (B <= 0 || n_kv_heads <= 0 || n_kv_heads > 8 || max_seq_len < 0 || kept < 0 || window < 0 ||
      steps_bound(max_seq_len, kept, window) <= kWholeSteps)
    return 0;
  return kept_workspace(n_kv_heads).total;
}

extern "C" int gkv_kept_decode(void *stream, int32_t B, int32_t n_q_heads, const float *q,
                               int64_t q_stride, const float *cos_tab, const float *sin_tab,
                               const int32_t *seq_lens, int32_t max_seq_len, gkv_cache_view cache,
                               int32_t kept, int32_t window, const float *sinks, void *workspace,
                               size_t workspace_bytes, void *out, int64_t out_stride,
                               int32_t out_dtype, uint32_t *dev_err) {
  using namespace gkv;
  if (B < 0 || n_q_heads <= 0 || max_seq_len < 0 || !q || !seq_lens || !out ||
      (out_dtype != GKV_F32 && out_dtype != GKV_BF16) || (cos_tab == nullptr) != (sin_tab == nullptr))
    return GKV_ERR_ARG;
  int st = kept_check(cache, kept, window, true);
  if (st != GKV_OK)
    return st;
  if (n_q_heads % cache.n_kv_heads != 0)
    return GKV_ERR_ARG;
  const int G = n_q_heads / cache.n_kv_heads;
  if (cache.n_kv_heads > 8 || G > kHeads)
    return GKV_ERR_UNSUPPORTED;
  if (q_stride < (int64_t)n_q_heads * kHeadDim || out_stride < (int64_t)n_q_heads * kHeadDim)
    return GKV_ERR_ARG;
  // 16-byte loads of the query rows and the angles, 16- (bf16: 8-) byte stores
  if (q_stride % 4 != 0 || out_stride % 4 != 0 ||
      ((uintptr_t)q | (uintptr_t)cos_tab | (uintptr_t)sin_tab) % 16 != 0 ||
      (uintptr_t)out % (out_dtype == GKV_BF16 ? 8 : 16) != 0)
    return GKV_ERR_ARG;
  const int64_t steps = steps_bound(max_seq_len, kept, window);
  if ((int64_t)B * steps >= INT32_MAX || (int64_t)B * cache.n_kv_heads >= INT32_MAX)
    return GKV_ERR_UNSUPPORTED; // 32-bit step counts
  const bool blk = cache.v_format == GKV_KV_FP8_BLOCK;
  KeptDecodeArgs a{};
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
  a.row = KeptRow{kept / kBlockTokens, cache.ring / kBlockTokens};
  a.window = window;
  a.max_len = (int)std::min<int64_t>(max_seq_len, kept_capacity(cache.table_stride, cache.ring) - 1);
  if (cache.ring == 0)
    a.max_len = (int)std::min<int64_t>(max_seq_len, kept_capacity(cache.table_stride, 0));
  a.sinks = sinks;
  a.B = B;
  a.G = G;
  a.n_kv_heads = cache.n_kv_heads;
  a.out = out;
  a.out_stride = out_stride;
  a.out_bf16 = out_dtype == GKV_BF16;
  a.dev_err = dev_err;
  hipStream_t s = (hipStream_t)stream;
  if (use_whole(B, a.n_kv_heads, max_seq_len, kept, window)) {
    if (B == 0)
      return GKV_OK;
    a.parts = whole_parts(B, a.n_kv_heads, steps, window);
    a.heads_per_wg = std::min(8 / a.parts, a.n_kv_heads);
    const int64_t wgs = (int64_t)B * ((a.n_kv_heads + a.heads_per_wg - 1) / a.heads_per_wg);
    const dim3 grid((unsigned)wgs), block(64 * a.parts * a.heads_per_wg);
    if (!grid_fits(wgs, block.x))
      return GKV_ERR_UNSUPPORTED;
    if (blk && a.out_bf16)
      hipLaunchKernelGGL((kept_decode_whole_kernel<true, 2, 4, false>), grid, block, 0, s, a);
    else if (blk)
      hipLaunchKernelGGL((kept_decode_whole_kernel<true, 2, 4, true>), grid, block, 0, s, a);
    else if (a.out_bf16)
      hipLaunchKernelGGL((kept_decode_whole_kernel<false, 2, 4, false>), grid, block, 0, s, a);
    else
      hipLaunchKernelGGL((kept_decode_whole_kernel<false, 2, 4, true>), grid, block, 0, s, a);
    return launch_status("kept_decode_whole_kernel");
  }
  const KeptWorkspace w = kept_workspace(a.n_kv_heads);
  if (B > 0 && (!workspace || workspace_bytes < w.total))
    return GKV_ERR_WORKSPACE;
  if ((uintptr_t)workspace % 16 != 0)
    return GKV_ERR_ARG;
  if (B == 0)
    return GKV_OK;
  const int subs = range_subs(a.n_kv_heads);
  a.max_ranges = kSplitWgs * subs;
  a.cuts = (int4 *)workspace;
  a.ws_ml = (float *)((char *)workspace + w.ml);
  a.ws_o = (float *)((char *)workspace + w.o);
  const dim3 block(64 * subs * a.n_kv_heads);
  if (blk && a.out_bf16)
    hipLaunchKernelGGL((kept_decode_split_kernel<true, 2, 2, false>), dim3(kSplitWgs), block, 0, s, a);
  else if (blk)
    hipLaunchKernelGGL((kept_decode_split_kernel<true, 2, 2, true>), dim3(kSplitWgs), block, 0, s, a);
  else if (a.out_bf16)
    hipLaunchKernelGGL((kept_decode_split_kernel<false, 2, 2, false>), dim3(kSplitWgs), block, 0, s, a);
  else
    hipLaunchKernelGGL((kept_decode_split_kernel<false, 2, 2, true>), dim3(kSplitWgs), block, 0, s, a);
  if ((st = launch_status("kept_decode_split_kernel")))
    return st;
  hipLaunchKernelGGL(kept_decode_merge_kernel, dim3((unsigned)a.max_ranges), dim3(kMergeThreads), 0, s,
                     a);
  return launch_status("kept_decode_merge_kernel");
}
