// Verification of drafted tokens (lmb200_verify_drafts).
//
// Row i of a sequence holds the target's logits behind its i-th token, and judges the next token t: with p = softmax(target / T) and
// q = softmax(draft / T) (without draft logits: all of q on t), t is taken where u q(t) < p(t).  The first row that takes nothing, or the last row, gives one new token:
// the smallest j with sum_{i <= j} w_i > u' sum w, w = max(p - q, 0), and w = p behind the last draft.  T <= 0: the largest logit judges and is given.
//
// Launches.  statistics_kernel reads every row once, split over CTAs, and leaves a maximum and a sum per part; decide_kernel joins the parts and finds the row that gives the token.
// That row is read again (it is in L2) with everything in 64 bits (exp64.cuh): where two borders of the running sum lie 1e-6 apart, sums of 32-bit exponentials, off by about 1e-8 of
// the total, would now and then choose the neighbour of the right token.  totals_kernel sums its exponentials over chunks of the vocabulary, weights_kernel the weights where they need
// those totals (max(p - q, 0)), and choose_kernel finds the chunk and in it the token.  at_once_kernel does the last four in one launch with a cluster per sequence: quicker for
// small vocabularies, slower for large ones, of which an SM gets two sequences or none.
#include <cooperative_groups.h>
#include <float.h>
#include <limits.h>
#include <math_constants.h>

#include <algorithm>

#include "exp64.cuh"
#include "kv4.cuh"
#include "pdl.cuh"

namespace lmb {
namespace {

constexpr int kStatThreads = 256, kChooseThreads = 512, kSplits = 16, kDecideThreads = 128, kMostChunks = 64, kChunk = 2048;
// Vocabularies up to this size take two launches, larger ones four or five.  One sequence of five rows: 32064 logits 15.5 against 16.9 us, 128256 39.7 against 22.9; 32 sequences: 32064
// 35.9 against 39.7, 128256 83 against 63.
constexpr int kAtOnce = 40960;

struct VerifyParams {
  const void *target, *draft;
  int64_t target_stride, draft_stride;
  int vocab, rows, n_seq, splits;
  const int *cu_rows, *tokens;
  const float *temperature, *accept_u, *sample_u;
  int *tokens_out, *n_out, *drop;
  int* dev_arg;
  int chunks;                                // of the vocabulary
  float4* part;                              // [rows][kSplits]: target's maximum and sum (T <= 0: the place of the maximum), draft's
  // of a sequence, at the place of its first row
  struct Choice* choice;                     // [rows]
  double2* total;                            // [rows][kMostChunks]: sums of the target's (without a token that is left out) and the draft's exponentials
  double* weight;                            // [rows][kMostChunks]
};

// a logit as it counts: NaN is no choice, infinities are the largest number
__device__ __forceinline__ float clean(float x) { return x == x ? fminf(x, FLT_MAX) : -CUDART_INF_F; }

// log2(e) / T, within what keeps 0 times it and -infinity times it defined
__device__ __forceinline__ float slope_of(float T) { return fminf(fmaxf(1.4426950408889634f / T, 1e-30f), 1e30f); }

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void join(float& m, float& s, float m2, float s2, float c) {
  const float mn = fmaxf(m, m2), mu = mn == -CUDART_INF_F ? 0.f : mn;
  s = s * exp2_fast((m - mu) * c) + s2 * exp2_fast((m2 - mu) * c);
  m = mn;
}
__device__ __forceinline__ void join_best(float& m, int& at, float m2, int at2) {
  if (m2 > m || (m2 == m && at2 < at && m > -CUDART_INF_F)) { m = m2; at = at2; }
}

// N neighbouring logits of a row from an aligned place
template <typename T> struct Run;
template <> struct Run<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void load(const float* p, float (&x)[4]) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(p));
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
  }
};
template <> struct Run<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void load(const __nv_bfloat16* p, float (&x)[8]) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};

// f(first, values) over this thread's share of part `split` of a row: aligned runs in the middle, kTogether of them at a time (-infinity where there is none), single values
// at the row's ends.
constexpr int kTogether = 4;
template <typename T, typename F>
__device__ __forceinline__ void walk(const T* row, int vocab, int split, int splits, F f) {
  constexpr int N = Run<T>::N;
  const int head = min(vocab, (int)((16 - ((uintptr_t)row & 15)) & 15) / (int)sizeof(T));
  const int runs = (vocab - head) / N, tail = head + runs * N;
  const int per = (runs + splits - 1) / splits, r1 = min(runs, (split + 1) * per);
  float x[kTogether][N];
  for (int r = split * per + (int)threadIdx.x; r < r1; r += kTogether * kStatThreads) {
#pragma unroll
    for (int h = 0; h < kTogether; ++h) {
      if (r + h * kStatThreads < r1) {
        Run<T>::load(row + head + (r + h * kStatThreads) * N, x[h]);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[h][i] = -CUDART_INF_F;
      }
    }
    f(head + r * N, x);
  }
  if (split == 0) {
    const int ends = head + (vocab - tail);
    for (int e = threadIdx.x; e < ends; e += kStatThreads) {
      const int j = e < head ? e : tail + (e - head);
#pragma unroll
      for (int h = 0; h < kTogether; ++h)
#pragma unroll
        for (int i = 0; i < N; ++i) x[h][i] = -CUDART_INF_F;
      x[0][0] = to_f32(row[j]);
      f(j, x);
    }
  }
}

// Maximum and sum of 2^(c (x - maximum)).  Values are taken as they are; where NaN or +infinity made the sum no number, the part is gone through again with every
// value cleaned.
template <typename T>
__device__ __forceinline__ float2 row_stats(const T* row, int vocab, int split, int splits, float c) {
  constexpr int N = Run<T>::N;
  float m, s;
  auto pass = [&](bool cleaned) {
    m = -CUDART_INF_F;
    s = 0.f;
    walk(row, vocab, split, splits, [&](int, float (&x)[kTogether][N]) {
      float top = -CUDART_INF_F;
#pragma unroll
      for (int h = 0; h < kTogether; ++h)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if (cleaned) x[h][i] = clean(x[h][i]);
          top = fmaxf(top, x[h][i]);
        }
      if (top > m) {
        s *= exp2_fast((m - top) * c);
        m = top;
      }
      const float mu = m == -CUDART_INF_F ? 0.f : m;
#pragma unroll
      for (int h = 0; h < kTogether; ++h) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) sum += exp2_fast((x[h][i] - mu) * c);        // (the difference first: T may be tiny)
        s += sum;
      }
    });
  };
  pass(false);
  if (!(s < CUDART_INF_F)) pass(true);
  __shared__ float2 red[kStatThreads / 32];
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) join(m, s, __shfl_xor_sync(0xffffffffu, m, off), __shfl_xor_sync(0xffffffffu, s, off), c);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_float2(m, s);
  __syncthreads();
  if (threadIdx.x >= 32) return make_float2(0.f, 0.f);       // the first warp's is asked for
  const float2 v = threadIdx.x < kStatThreads / 32 ? red[threadIdx.x] : make_float2(-CUDART_INF_F, 0.f);
  m = v.x;
  s = v.y;
#pragma unroll
  for (int off = kStatThreads / 64; off > 0; off >>= 1) join(m, s, __shfl_xor_sync(0xffffffffu, m, off), __shfl_xor_sync(0xffffffffu, s, off), c);
  return make_float2(m, s);
}

// the sequence of a row: the last b with cu[b] <= row and rows of its own; -1 where there is none
__device__ __forceinline__ int sequence_of(const int* cu, int n_seq, int row) {
  int lo = 0, hi = n_seq;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid + 1] <= row) lo = mid + 1; else hi = mid;
  }
  return lo < n_seq && cu[lo] <= row ? lo : -1;
}

template <typename T>
__global__ void __launch_bounds__(kStatThreads) statistics_kernel(const VerifyParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.y, split = blockIdx.x;
  const int b = sequence_of(p.cu_rows, p.n_seq, row);
  if (b < 0) return;
  const float temperature = p.temperature ? p.temperature[b] : 0.f;
  const T* target = reinterpret_cast<const T*>(p.target) + row * p.target_stride;
  float4 out = make_float4(0.f, 0.f, -CUDART_INF_F, 0.f);
  if (temperature > 0.f) {
    const float c = slope_of(temperature);
    const float2 a = row_stats(target, p.vocab, split, p.splits, c);
    out.x = a.x;
    out.y = a.y;
    if (p.draft && row + 1 < p.cu_rows[b + 1]) {                       // the last row judges no draft
      const float2 d = row_stats(reinterpret_cast<const T*>(p.draft) + row * p.draft_stride, p.vocab, split, p.splits, c);
      out.z = d.x;
      out.w = d.y;
    }
  } else {
    float m = -CUDART_INF_F;
    int at = INT_MAX;
    walk(target, p.vocab, split, p.splits, [&](int first, float (&x)[kTogether][Run<T>::N]) {
#pragma unroll
      for (int h = 0; h < kTogether; ++h) {
        float top = x[h][0];
#pragma unroll
        for (int i = 1; i < Run<T>::N; ++i) top = fmaxf(top, x[h][i]);
        if (top > -CUDART_INF_F && top >= m) {               // a new maximum, or an equal one
#pragma unroll
          for (int i = 0; i < Run<T>::N; ++i) join_best(m, at, clean(x[h][i]), first + h * kStatThreads * Run<T>::N + i);
        }
      }
    });
    __shared__ float2 red[kStatThreads / 32];
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) join_best(m, at, __shfl_xor_sync(0xffffffffu, m, off), __shfl_xor_sync(0xffffffffu, at, off));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_float2(m, __int_as_float(at));
    __syncthreads();
    for (int w = 0; w < kStatThreads / 32; ++w) join_best(m, at, red[w].x, __float_as_int(red[w].y));
    out.x = m;
    out.y = __int_as_float(at);
  }
  if (threadIdx.x == 0) p.part[(int64_t)row * kSplits + split] = out;
}

// What a sequence's token is chosen from.
struct Choice {
  int row;                                   // -1: the token is there
  int without;                               // token that is left out, or -1
  int minus;                                 // the draft's probabilities are taken off
  float top, draft_top;
};

// A chunk of the chosen row: thread's runs of N neighbouring logits, of the target and the draft.
template <typename T> struct Chunk {
  static constexpr int N = Run<T>::N;
  const T *target, *draft;
  int first, end, vocab;                     // runs
  bool aligned, minus;
  __device__ __forceinline__ Chunk(const VerifyParams& p, const Choice& c, int chunk)
      : target(reinterpret_cast<const T*>(p.target) + c.row * p.target_stride), draft(reinterpret_cast<const T*>(p.draft) + c.row * p.draft_stride), vocab(p.vocab), minus(c.minus) {
    const int runs = (p.vocab + N - 1) / N, per = (runs + p.chunks - 1) / p.chunks;
    first = min(runs, chunk * per);
    end = min(runs, first + per);
    aligned = (((uintptr_t)target | (minus ? (uintptr_t)draft : 0)) & 15) == 0;
  }
  __device__ __forceinline__ void load(int run, float (&a)[N], float (&d)[N]) const {
    const int j = run * N;
    if (aligned && run < end && j + N <= vocab) {
      Run<T>::load(target + j, a);
      if (minus) Run<T>::load(draft + j, d);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const bool there = run < end && j + i < vocab;
        a[i] = there ? to_f32(target[j + i]) : -CUDART_INF_F;
        if (minus) d[i] = there ? to_f32(draft[j + i]) : -CUDART_INF_F;
      }
    }
  }
};

// The weights of a run's tokens.
template <int N>
__device__ __forceinline__ void weights_of(const Power& ep, const Power& eq, bool minus, double ip, double iq, int without, int first, const float (&a)[N], const float (&d)[N],
                                           double (&w)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    w[i] = ep(a[i]);
    if (minus) {                             // (products rounded, so 0 where the two are equal)
      const double x = __dsub_rn(__dmul_rn(w[i], ip), __dmul_rn(eq(d[i]), iq));
      w[i] = x > 0.0 ? x : 0.0;
    } else if (first + i == without) {
      w[i] = 0.0;
    }
  }
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}
template <int kThreads> __device__ __forceinline__ double block_sum(double v, double* red) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
  for (int w = 0; w < kThreads / 32; ++w) s += red[w];
  return s;
}
// a sequence's first row; -1: it has none, or rows that are not there
__device__ __forceinline__ int first_row(const VerifyParams& p, int b) {
  const int r0 = p.cu_rows[b], r1 = p.cu_rows[b + 1];
  return r0 < 0 || r1 > p.rows || r1 <= r0 ? -1 : r0;
}
__device__ __forceinline__ double inverse_T(const VerifyParams& p, int b) { return fmin(fmax(1.0 / (double)p.temperature[b], 1e-30), 1e30); }

// A block finds out which drafts of sequence b (rows r0 to r1 - 1) are taken, and what the next token is chosen from (by all threads known at the end); `writes`: and writes
// down what is known.  A warp per row.
template <typename T, int kThreads>
__device__ __forceinline__ Choice decide(const VerifyParams& p, int b, int r0, int r1, bool writes) {
  constexpr int kWarps = kThreads / 32;
  __shared__ int stop_row;
  __shared__ Choice found;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) stop_row = r1 - 1;
  const float temperature = p.temperature ? p.temperature[b] : 0.f;
  const bool greedy = !(temperature > 0.f);
  const double slope = greedy ? 1.0 : inverse_T(p, b) * 1.4426950408889634;
  __syncthreads();
  // the parts of a row, joined by a warp; a refused draft ends the sequence there
  auto joined = [&](int row, float& m, double& s, float& md, double& sd) {
    const float4 v = lane < p.splits ? p.part[(int64_t)row * kSplits + lane] : make_float4(-CUDART_INF_F, 0.f, -CUDART_INF_F, 0.f);
    m = v.x;
    md = v.z;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
      md = fmaxf(md, __shfl_xor_sync(0xffffffffu, md, off));
    }
    s = warp_sum(v.x == -CUDART_INF_F ? 0.0 : (double)v.y * exp2(((double)v.x - m) * slope));
    sd = warp_sum(v.z == -CUDART_INF_F ? 0.0 : (double)v.w * exp2(((double)v.z - md) * slope));
  };
  auto best_of = [&](int row, float& m) {
    const float4 v = lane < p.splits ? p.part[(int64_t)row * kSplits + lane] : make_float4(-CUDART_INF_F, __int_as_float(INT_MAX), 0.f, 0.f);
    m = v.x;
    int at = __float_as_int(v.y);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) join_best(m, at, __shfl_xor_sync(0xffffffffu, m, off), __shfl_xor_sync(0xffffffffu, at, off));
    return at;
  };
  auto logit = [&](const void* base, int64_t stride, int row, int j) { return clean(to_f32(reinterpret_cast<const T*>(base)[row * stride + j])); };
  for (int row = r0 + warp; row < r1 - 1; row += kWarps) {
    const int t = p.tokens[row + 1];
    bool takes;
    if (greedy) {
      float m;
      takes = best_of(row, m) == t && m > -CUDART_INF_F;
    } else {
      float m, md;
      double s, sd;
      const bool known = t >= 0 && t < p.vocab;
      const float l = known ? logit(p.target, p.target_stride, row, t) : -CUDART_INF_F, ld = known && p.draft ? logit(p.draft, p.draft_stride, row, t) : -CUDART_INF_F;
      joined(row, m, s, md, sd);
      const double pt = l == -CUDART_INF_F ? 0.0 : exp2(((double)l - m) * slope) / s;
      const double qt = !p.draft ? 1.0 : ld == -CUDART_INF_F ? 0.0 : exp2(((double)ld - md) * slope) / sd;
      takes = (double)p.accept_u[row] * qt < pt;
    }
    if (lane == 0 && !takes) atomicMin(&stop_row, row);
  }
  __syncthreads();
  const int stop = stop_row;
  if (warp == 0) {
    Choice c = {stop, -1, 0, -CUDART_INF_F, -CUDART_INF_F};
    int token = -1;
    if (greedy) {
      const int at = best_of(stop, c.top);
      if (c.top > -CUDART_INF_F && (unsigned)at < (unsigned)p.vocab) token = at;       // (rows that offsets give to two sequences may have no statistics)
      c.row = -1;
    } else {
      double s, sd;
      joined(stop, c.top, s, c.draft_top, sd);
      const bool last = stop == r1 - 1;
      c.minus = !last && p.draft && c.draft_top > -CUDART_INF_F;
      if (!last && !p.draft) c.without = p.tokens[stop + 1];
      if (c.top == -CUDART_INF_F) c.row = -1;                // nothing can be chosen
    }
    if (lane == 0) {
      found = c;
      if (writes) {
        if (c.row < 0) p.tokens_out[stop] = token;
        p.n_out[b] = stop - r0 + 1;
        p.drop[b] = r1 - 1 - stop;
      }
    }
  }
  for (int row = r0 + tid; writes && row < r1; row += kThreads)
    if (row != stop) p.tokens_out[row] = row < stop ? p.tokens[row + 1] : -1;
  __syncthreads();
  return found;
}

// A sequence without rows, or with rows that are not there.
__device__ __forceinline__ void no_rows(const VerifyParams& p, int b) {
  if (threadIdx.x) return;
  p.n_out[b] = 0;
  p.drop[b] = 0;
  if (p.cu_rows[b + 1] != p.cu_rows[b]) atomicExch(p.dev_arg, kv4::kErrPage);
}

// One CTA per sequence.
template <typename T>
__global__ void __launch_bounds__(kDecideThreads) decide_kernel(const VerifyParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.x, r0 = first_row(p, b);
  if (r0 < 0) return no_rows(p, b);
  const Choice c = decide<T, kDecideThreads>(p, b, r0, p.cu_rows[b + 1], true);
  if (threadIdx.x == 0) p.choice[r0] = c;
}

// Sums of the exponentials of a chunk, the whole block's: target's (without a token that is left out) and draft's.
template <typename T, int kThreads>
__device__ __forceinline__ double2 totals_in(const Chunk<T>& chunk_of, const Choice& c, const Power& ep, const Power& eq, double* red) {
  constexpr int N = Run<T>::N;
  double sp = 0.0, sq = 0.0;
  for (int run = chunk_of.first + (int)threadIdx.x; run < chunk_of.end; run += 2 * kThreads) {
    float a[2][N], d[2][N];
#pragma unroll
    for (int h = 0; h < 2; ++h) chunk_of.load(run + h * kThreads, a[h], d[h]);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const double e = ep(a[h][i]);
        if (c.minus) sq += eq(d[h][i]);
        if ((run + h * kThreads) * N + i != c.without) sp += e;
      }
  }
  sp = block_sum<kThreads>(sp, red);
  if (c.minus) sq = block_sum<kThreads>(sq, red);
  return make_double2(sp, sq);
}

// Sum of the weights max(p - q, 0) of a chunk.
template <typename T, int kThreads>
__device__ __forceinline__ double weights_in(const Chunk<T>& chunk_of, const Power& ep, const Power& eq, double ip, double iq, double* red) {
  constexpr int N = Run<T>::N;
  double sum = 0.0;
  for (int run = chunk_of.first + (int)threadIdx.x; run < chunk_of.end; run += kThreads) {
    float a[N], d[N];
    double w[N];
    chunk_of.load(run, a, d);
    weights_of<N>(ep, eq, true, ip, iq, -1, run * N, a, d, w);
#pragma unroll
    for (int i = 0; i < N; ++i) sum += w[i];
  }
  return block_sum<kThreads>(sum, red);
}

// Of up to 64 neighbouring sums, two per lane, the first at which the running sum passes the goal; by rounding there may be none, then the last above 0.  `before`: the sums in front of it.
__device__ __forceinline__ int passing_part(double v0, double v1, double goal, double& before) {
  const int lane = threadIdx.x & 31;
  before = v0 + v1;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const double x = __shfl_up_sync(0xffffffffu, before, off);
    if (lane >= off) before += x;
  }
  const unsigned passing = __ballot_sync(0xffffffffu, v0 + v1 > 0.0 && before > goal), having = __ballot_sync(0xffffffffu, v0 + v1 > 0.0);
  const int who = passing ? __ffs(passing) - 1 : 31 - __clz(having);
  before -= v0 + v1;
  int part = 2 * lane;
  if (!(v0 > 0.0) || (v1 > 0.0 && !(before + v0 > goal))) { before += v0; ++part; }
  before = __shfl_sync(0xffffffffu, before, who);
  return __shfl_sync(0xffffffffu, part, who);
}

// The token of a chunk at which the running sum, `before` in front of the chunk, passes the goal, or the last with any weight.
template <typename T, int kThreads>
__device__ __forceinline__ void find_token(const VerifyParams& p, const Chunk<T>& chunk_of, const Choice& c, const Power& ep, const Power& eq, double ip, double iq, double before,
                                           double goal) {
  constexpr int kWarps = kThreads / 32, N = Run<T>::N;
  __shared__ double of_warp[kWarps];
  __shared__ int token, first_pass, last_some;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) token = -1;
  for (int base = chunk_of.first; base < chunk_of.end; base += kThreads) {
    const int run = base + tid;
    float a[N], d[N];
    double w[N], v = 0.0;
    chunk_of.load(run, a, d);
    weights_of<N>(ep, eq, c.minus, ip, iq, c.without, run * N, a, d, w);
#pragma unroll
    for (int i = 0; i < N; ++i) v += w[i];
    double incl = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const double x = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += x;
    }
    __syncthreads();
    if (lane == 31) of_warp[warp] = incl;
    __syncthreads();
    double mine = before + incl - v;         // in front of this run
    for (int k = 0; k < warp; ++k) mine += of_warp[k];
    for (int k = 0; k < kWarps; ++k) before += of_warp[k];
    // the first run that passes has the token; without one the last run with any weight, so far
    const bool passes = v > 0.0 && mine + v > goal;
    if (tid == 0) { first_pass = INT_MAX; last_some = -1; }
    __syncthreads();
    if (passes) atomicMin(&first_pass, run);
    if (v > 0.0) atomicMax(&last_some, run);
    __syncthreads();
    if (run == (first_pass != INT_MAX ? first_pass : last_some)) {
      bool done = false;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        mine += w[i];
        if (w[i] > 0.0 && !done) { token = run * N + i; done = mine > goal; }
      }
    }
    if (first_pass != INT_MAX) break;
  }
  __syncthreads();
  if (tid == 0) p.tokens_out[c.row] = token;
}

template <typename T>
__global__ void __launch_bounds__(kStatThreads) totals_kernel(const VerifyParams p) {
  __shared__ double red[kStatThreads / 32], table[32];
  fill_table(table);
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x;
  const int r0 = first_row(p, b);
  if (r0 < 0) return;
  const Choice c = p.choice[r0];
  if (c.row < 0) return;
  const double inv_T = inverse_T(p, b);
  __syncthreads();
  const double2 t = totals_in<T, kStatThreads>(Chunk<T>(p, c, chunk), c, Power(table, c.top, inv_T), Power(table, c.minus ? c.draft_top : 0.f, inv_T), red);
  if (tid == 0) p.total[(int64_t)r0 * kMostChunks + chunk] = t;
}

// sums over a sequence's chunks, by a whole warp
__device__ __forceinline__ double2 totals_of(const VerifyParams& p, int r0) {
  double sp = 0.0, sq = 0.0;
  for (int k = threadIdx.x & 31; k < p.chunks; k += 32) {
    const double2 v = p.total[(int64_t)r0 * kMostChunks + k];
    sp += v.x;
    sq += v.y;
  }
  return make_double2(warp_sum(sp), warp_sum(sq));
}

template <typename T>
__global__ void __launch_bounds__(kStatThreads) weights_kernel(const VerifyParams p) {
  __shared__ double red[kStatThreads / 32], table[32];
  fill_table(table);
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.y, chunk = blockIdx.x;
  const int r0 = first_row(p, b);
  if (r0 < 0) return;
  const Choice c = p.choice[r0];
  if (c.row < 0 || !c.minus) return;         // else the totals are the weights' own
  const double inv_T = inverse_T(p, b);
  const double2 total = totals_of(p, r0);
  __syncthreads();
  const double w = weights_in<T, kStatThreads>(Chunk<T>(p, c, chunk), Power(table, c.top, inv_T), Power(table, c.draft_top, inv_T), 1.0 / total.x, 1.0 / total.y, red);
  if (threadIdx.x == 0) p.weight[(int64_t)r0 * kMostChunks + chunk] = w;
}

// One CTA per sequence: the chunk in which the running sum passes its goal, then the token.
template <typename T>
__global__ void __launch_bounds__(kChooseThreads) choose_kernel(const VerifyParams p) {
  __shared__ double table[32];
  fill_table(table);
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.x, lane = threadIdx.x & 31;
  const int r0 = first_row(p, b);
  if (r0 < 0) return;
  Choice c = p.choice[r0];
  if (c.row < 0) return;
  const double inv_T = inverse_T(p, b);
  const double2 total = totals_of(p, r0);
  static_assert(kMostChunks == 64, "two chunks a lane");
  double v0, v1, sum;
  for (bool again = false;; again = true) {  // p <= q everywhere: the target itself
    auto at = [&](int k) { return k >= p.chunks ? 0.0 : c.minus ? p.weight[(int64_t)r0 * kMostChunks + k] : p.total[(int64_t)r0 * kMostChunks + k].x; };
    v0 = at(2 * lane);
    v1 = at(2 * lane + 1);
    sum = warp_sum(v0 + v1);
    if (sum > 0.0 || again || !c.minus) break;
    c.minus = 0;
  }
  if (!(sum > 0.0)) {                        // nothing but the refused draft
    if (threadIdx.x == 0) p.tokens_out[c.row] = c.without;
    return;
  }
  const double goal = (double)p.sample_u[b] * sum;
  double before;
  const int chunk = passing_part(v0, v1, goal, before);
  __syncthreads();                           // the table
  find_token<T, kChooseThreads>(p, Chunk<T>(p, c, chunk), c, Power(table, c.top, inv_T), Power(table, c.minus ? c.draft_top : 0.f, inv_T), 1.0 / total.x, 1.0 / total.y, before, goal);
}

// All of that in one launch, a cluster per sequence and a CTA per chunk: where there is little to do, the launches are what it takes.
template <typename T>
__global__ void __launch_bounds__(kChooseThreads) at_once_kernel(const VerifyParams p) {
  namespace cg = cooperative_groups;
  __shared__ double red[kChooseThreads / 32], table[32], mine[4];        // this CTA's sums, read by its cluster
  fill_table(table);
  pdl_launch_dependents();
  pdl_wait();
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), b = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31;
  const int r0 = first_row(p, b);
  if (r0 < 0) {                              // the same for the whole cluster, as every return before its last barrier
    if (rank == 0) no_rows(p, b);
    return;
  }
  Choice c = decide<T, kChooseThreads>(p, b, r0, p.cu_rows[b + 1], rank == 0);
  if (c.row < 0) return;
  const double inv_T = inverse_T(p, b);
  const Chunk<T> chunk_of(p, c, rank);
  const Power ep(table, c.top, inv_T), eq(table, c.minus ? c.draft_top : 0.f, inv_T);
  const double2 t = totals_in<T, kChooseThreads>(chunk_of, c, ep, eq, red);
  if (tid == 0) { mine[0] = t.x; mine[1] = t.y; }
  cluster.sync();
  auto of = [&](int what, int k) { return k < C ? *cluster.map_shared_rank(mine + what, k) : 0.0; };
  const double sp = warp_sum(of(0, lane)), sq = warp_sum(of(1, lane));
  const double ip = 1.0 / sp, iq = 1.0 / sq;
  double v0 = of(0, 2 * lane), v1 = of(0, 2 * lane + 1), sum = sp;
  if (c.minus) {
    const double w = weights_in<T, kChooseThreads>(chunk_of, ep, eq, ip, iq, red);
    if (tid == 0) mine[2] = w;
    cluster.sync();
    const double s = warp_sum(of(2, lane));
    if (s > 0.0) { sum = s; v0 = of(2, 2 * lane); v1 = of(2, 2 * lane + 1); }
    else c.minus = 0;                        // p <= q everywhere: the target itself
  }
  cluster.sync();                            // no CTA leaves while others read its sums
  if (!(sum > 0.0)) {                        // nothing but the refused draft
    if (rank == 0 && tid == 0) p.tokens_out[c.row] = c.without;
    return;
  }
  const double goal = (double)p.sample_u[b] * sum;
  double before;
  if (passing_part(v0, v1, goal, before) != rank) return;
  find_token<T, kChooseThreads>(p, Chunk<T>(p, c, rank), c, ep, eq, ip, iq, before, goal);
}

template <typename T>
int32_t launch_verify(Ctx* ctx, const VerifyParams& p) {
  LMB_CUDA(launch_k_opt(false, statistics_kernel<T>, dim3((unsigned)p.splits, (unsigned)p.rows), dim3(kStatThreads), 0, ctx->stream, p));
  ctx->launches++;
  if (p.vocab <= kAtOnce) {
    VerifyParams q = p;
    q.chunks = p.vocab <= 4096 ? 1 : 8;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(q.n_seq * q.chunks));
    cfg.blockDim = dim3(kChooseThreads);
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)q.chunks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    LMB_CUDA(cudaLaunchKernelEx(&cfg, at_once_kernel<T>, q));
    ctx->launches++;
    return LMB200_OK;
  }
  const dim3 grid((unsigned)p.chunks, (unsigned)p.n_seq);
  LMB_CUDA(launch_k(decide_kernel<T>, dim3((unsigned)p.n_seq), dim3(kDecideThreads), 0, ctx->stream, p));
  ctx->launches++;
  if (!p.temperature) return LMB200_OK;      // the tokens are there
  LMB_CUDA(launch_k(totals_kernel<T>, grid, dim3(kStatThreads), 0, ctx->stream, p));
  ctx->launches++;
  if (p.draft) {
    LMB_CUDA(launch_k(weights_kernel<T>, grid, dim3(kStatThreads), 0, ctx->stream, p));
    ctx->launches++;
  }
  LMB_CUDA(launch_k(choose_kernel<T>, dim3((unsigned)p.n_seq), dim3(kChooseThreads), 0, ctx->stream, p));
  ctx->launches++;
  return LMB200_OK;
}

}  // namespace
}  // namespace lmb

using namespace lmb;

// A sequence that has work has a row, so its place in the workspace is its first row's.
extern "C" int32_t lmb200_verify_drafts_workspace(int32_t rows, int64_t* bytes) {
  LMB_REQUIRE(bytes && rows >= 0, "verify_drafts_workspace: bad argument");
  *bytes = std::max<int64_t>(16, (int64_t)rows * (kSplits * sizeof(float4) + kMostChunks * (sizeof(double2) + sizeof(double)) + 32));
  return LMB200_OK;
}

extern "C" int32_t lmb200_verify_drafts(lmb200_ctx h, int32_t dtype, const void* target, int64_t target_stride, const void* draft, int64_t draft_stride, int32_t vocab,
                                        int32_t rows, int32_t n_seq, const int32_t* cu_rows, const int32_t* tokens, const float* temperature, const float* accept_u,
                                        const float* sample_u, int32_t* tokens_out, int32_t* n_out, int32_t* drop, void* workspace, int64_t workspace_bytes) {
  Ctx* ctx = ctx_from(h);
  if (!ctx) return LMB200_EINVAL;
  LMB_REQUIRE(dtype == LMB200_F32 || dtype == LMB200_BF16, "verify_drafts: dtype %d", dtype);
  LMB_REQUIRE(vocab >= 1 && vocab <= (1 << 30), "verify_drafts: vocabulary of %d", vocab);
  LMB_REQUIRE(rows >= 0 && rows <= 65535 && n_seq >= 1 && n_seq <= 65535, "verify_drafts: %d rows (up to 65535) of %d sequences (1 to 65535)", rows, n_seq);
  LMB_REQUIRE(cu_rows && n_out && drop && (rows == 0 || (target && tokens && tokens_out && workspace)), "verify_drafts: null pointer");
  LMB_REQUIRE(!temperature || (accept_u && sample_u) || rows == 0, "verify_drafts: temperatures without random numbers");
  LMB_REQUIRE(target_stride >= vocab && (!draft || draft_stride >= vocab), "verify_drafts: row strides %lld and %lld for %d logits", (long long)target_stride,
              (long long)draft_stride, vocab);
  const uintptr_t size1 = dtype == LMB200_F32 ? 3 : 1;
  LMB_REQUIRE(((uintptr_t)target & size1) == 0 && ((uintptr_t)draft & size1) == 0 && (uintptr_t)workspace % 16 == 0,
              "verify_drafts: logits must start on a multiple of their size, the workspace on 16 bytes");
  int64_t need = 0;
  LMB_TRY(lmb200_verify_drafts_workspace(rows, &need));
  LMB_REQUIRE(rows == 0 || workspace_bytes >= need, "verify_drafts: a workspace of %lld bytes, %lld are needed", (long long)workspace_bytes, (long long)need);
  LMB_REQUIRE(rows == 0 || tokens_out != tokens, "verify_drafts: tokens_out may not be tokens");
  LMB_CUDA(cudaSetDevice(ctx->device));
  if (rows == 0) {
    LMB_CUDA(cudaMemsetAsync(n_out, 0, (size_t)n_seq * 4, ctx->stream));
    LMB_CUDA(cudaMemsetAsync(drop, 0, (size_t)n_seq * 4, ctx->stream));
    return LMB200_OK;
  }
  VerifyParams p = {target, draft, target_stride, draft_stride, vocab, rows, n_seq, vocab <= 4096 ? 1 : kSplits, cu_rows, tokens, temperature, accept_u, sample_u,
                    tokens_out, n_out, drop, ctx->dev_arg, (int)std::min<int64_t>(kMostChunks, ceil_div(vocab, kChunk))};
  p.part = static_cast<float4*>(workspace);
  p.total = reinterpret_cast<double2*>(p.part + (int64_t)rows * kSplits);
  p.weight = reinterpret_cast<double*>(p.total + (int64_t)rows * kMostChunks);
  p.choice = reinterpret_cast<Choice*>(p.weight + (int64_t)rows * kMostChunks);
  return dtype == LMB200_F32 ? launch_verify<float>(ctx, p) : launch_verify<__nv_bfloat16>(ctx, p);
}
