// Verification of drafted tokens (lmb200_verify_drafts).
//
// Row i of a sequence holds the target's logits behind its i-th token, and judges the next token t: with p = softmax(target / T) and
// q = softmax(draft / T) (without draft logits: all of q on t), t is taken where u q(t) < p(t).  The first row that takes nothing, or the last row, gives one new token:
// the smallest j with sum_{i <= j} w_i > u' sum w, w = max(p - q, 0), and w = p behind the last draft.  T <= 0: the largest logit judges and is given.
//
// Two launches.  statistics_kernel reads every row once, split over CTAs, and leaves a maximum and a sum per part.  choose_kernel, a cluster per sequence, joins the parts,
// finds the row that gives the token and reads that row again (it is in L2) for the sums in 64 bits: where two borders of the running sum lie 1e-6 apart, sums of 32-bit
// exponentials, off by about 1e-8 of the total, would now and then choose the neighbour of the right token.
#include <cooperative_groups.h>
#include <float.h>
#include <limits.h>
#include <math_constants.h>

#include <algorithm>

#include "kv4.cuh"
#include "pdl.cuh"

namespace lmb {
namespace {

constexpr int kStatThreads = 256, kChooseThreads = 512, kSplits = 16;

struct VerifyParams {
  const void *target, *draft;
  int64_t target_stride, draft_stride;
  int vocab, rows, n_seq, splits;
  const int *cu_rows, *tokens;
  const float *temperature, *accept_u, *sample_u;
  int *tokens_out, *n_out, *drop;
  int* dev_err;
  float4* part;                              // [rows][kSplits]: target's maximum and sum (or the place of the maximum), draft's
};

// a logit as it counts: NaN is no choice, infinities are the largest number
__device__ __forceinline__ float clean(float x) { return x == x ? fminf(x, FLT_MAX) : -CUDART_INF_F; }

// log2(e) / T, within what keeps 0 times it and -infinity times it defined
__device__ __forceinline__ float slope_of(float T) { return fminf(fmaxf(1.4426950408889634f / T, 1e-30f), 1e30f); }

__device__ __forceinline__ void join(float& m, float& s, float m2, float s2, float c) {
  const float mn = fmaxf(m, m2), mu = mn == -CUDART_INF_F ? 0.f : mn;
  s = s * exp2f((m - mu) * c) + s2 * exp2f((m2 - mu) * c);
  m = mn;
}
__device__ __forceinline__ void join_best(float& m, int& at, float m2, int at2) {
  if (m2 > m || (m2 == m && at2 < at)) { m = m2; at = at2; }
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

// f(first, values, count) over this thread's share of part `split` of a row: aligned runs in the middle, single values at the row's ends.
template <typename T, typename F>
__device__ __forceinline__ void walk(const T* row, int vocab, int split, int splits, F f) {
  constexpr int N = Run<T>::N;
  const int head = min(vocab, (int)((16 - ((uintptr_t)row & 15)) & 15) / (int)sizeof(T));
  const int runs = (vocab - head) / N, tail = head + runs * N;
  const int per = (runs + splits - 1) / splits, r1 = min(runs, (split + 1) * per);
  float x[N];
#pragma unroll 2
  for (int r = split * per + (int)threadIdx.x; r < r1; r += blockDim.x) {
    Run<T>::load(row + head + r * N, x);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = clean(x[i]);
    f(head + r * N, x, N);
  }
  if (split == 0) {
    const int ends = head + (vocab - tail);
    for (int e = threadIdx.x; e < ends; e += blockDim.x) {
      const int j = e < head ? e : tail + (e - head);
      x[0] = clean(to_f32(row[j]));
#pragma unroll
      for (int i = 1; i < N; ++i) x[i] = -CUDART_INF_F;
      f(j, x, 1);
    }
  }
}

template <typename T>
__device__ __forceinline__ float2 row_stats(const T* row, int vocab, int split, int splits, float c) {
  float m = -CUDART_INF_F, s = 0.f;
  walk(row, vocab, split, splits, [&](int, const float* x, int) {
    float top = x[0];
#pragma unroll
    for (int i = 1; i < Run<T>::N; ++i) top = fmaxf(top, x[i]);
    const float mn = fmaxf(m, top), mu = mn == -CUDART_INF_F ? 0.f : mn;
    s *= exp2f((m - mu) * c);
#pragma unroll
    for (int i = 0; i < Run<T>::N; ++i) s += exp2f((x[i] - mu) * c);
    m = mn;
  });
  __shared__ float2 red[kStatThreads / 32];
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) join(m, s, __shfl_xor_sync(0xffffffffu, m, off), __shfl_xor_sync(0xffffffffu, s, off), c);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_float2(m, s);
  __syncthreads();
  for (int w = 0; w < kStatThreads / 32; ++w)
    if (w != (int)(threadIdx.x >> 5)) join(m, s, red[w].x, red[w].y, c);
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
    walk(target, p.vocab, split, p.splits, [&](int first, const float* x, int) {
#pragma unroll
      for (int i = 0; i < Run<T>::N; ++i)
        if (x[i] > m || (x[i] == m && x[i] > -CUDART_INF_F && first + i < at)) { m = x[i]; at = first + i; }
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

__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
  for (int w = 0; w < kChooseThreads / 32; ++w) s += red[w];
  return s;
}

template <typename T>
__global__ void __launch_bounds__(kChooseThreads) choose_kernel(const VerifyParams p) {
  namespace cg = cooperative_groups;
  constexpr int kWarps = kChooseThreads / 32;
  __shared__ int stop_row;
  __shared__ double red[kWarps], of_warp[kWarps];
  __shared__ double cta[4];                  // this CTA's sums, read by its cluster
  pdl_launch_dependents();
  pdl_wait();
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int b = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r0 = p.cu_rows[b], r1 = p.cu_rows[b + 1];
  if (r0 < 0 || r1 > p.rows || r1 <= r0) {   // no row of its own, or rows that are not there: the same for the whole cluster
    if (rank == 0 && tid == 0) {
      p.n_out[b] = 0;
      p.drop[b] = 0;
      if (r1 != r0) atomicExch(p.dev_err, kv4::kErrPage);
    }
    return;
  }
  const float temperature = p.temperature ? p.temperature[b] : 0.f;
  const bool greedy = !(temperature > 0.f);
  const double inv_T = greedy ? 1.0 : fmin(fmax(1.0 / (double)temperature, 1e-30), 1e30);
  if (tid == 0) stop_row = r1 - 1;
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
    s = v.x == -CUDART_INF_F ? 0.0 : (double)v.y * exp(((double)v.x - m) * inv_T);
    sd = v.z == -CUDART_INF_F ? 0.0 : (double)v.w * exp(((double)v.z - md) * inv_T);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, off);
      sd += __shfl_xor_sync(0xffffffffu, sd, off);
    }
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
      joined(row, m, s, md, sd);
      const bool known = t >= 0 && t < p.vocab;
      const float l = known ? logit(p.target, p.target_stride, row, t) : -CUDART_INF_F;
      const double pt = l == -CUDART_INF_F ? 0.0 : exp(((double)l - m) * inv_T) / s;
      double qt = 1.0;
      if (p.draft) {
        const float ld = known ? logit(p.draft, p.draft_stride, row, t) : -CUDART_INF_F;
        qt = ld == -CUDART_INF_F ? 0.0 : exp(((double)ld - md) * inv_T) / sd;
      }
      takes = (double)p.accept_u[row] * qt < pt;
    }
    if (lane == 0 && !takes) atomicMin(&stop_row, row);
  }
  __syncthreads();
  const int stop = stop_row;
  if (rank == 0) {
    for (int row = r0 + tid; row < r1; row += kChooseThreads)
      if (row != stop) p.tokens_out[row] = row < stop ? p.tokens[row + 1] : -1;
    if (tid == 0) { p.n_out[b] = stop - r0 + 1; p.drop[b] = r1 - 1 - stop; }
  }
  if (greedy) {
    if (rank == 0 && warp == 0) {
      float m;
      const int at = best_of(stop, m);
      if (lane == 0) p.tokens_out[stop] = m > -CUDART_INF_F ? at : -1;
    }
    return;
  }
  float m, md;
  double s32, sd32;
  joined(stop, m, s32, md, sd32);
  if (m == -CUDART_INF_F) {                  // nothing can be chosen
    if (rank == 0 && tid == 0) p.tokens_out[stop] = -1;
    return;
  }
  const bool last = stop == r1 - 1;
  bool minus = !last && p.draft && md > -CUDART_INF_F;
  const int without = !last && !p.draft ? p.tokens[stop + 1] : -1;
  const T* target = reinterpret_cast<const T*>(p.target) + stop * p.target_stride;
  const T* draft = reinterpret_cast<const T*>(p.draft) + stop * p.draft_stride;
  // CTA `rank` has the tokens [first, end), a warp neighbours among them, a lane neighbours among those
  const int per_cta = (p.vocab + C - 1) / C, per_warp = (per_cta + kWarps - 1) / kWarps;
  const int c0 = min(p.vocab, rank * per_cta), c1 = min(p.vocab, c0 + per_cta);
  const int w0 = min(c1, c0 + warp * per_warp), w1 = min(c1, w0 + per_warp);
  auto ep = [&](int j) { return exp(((double)clean(to_f32(target[j])) - m) * inv_T); };
  auto eq = [&](int j) { return exp(((double)clean(to_f32(draft[j])) - md) * inv_T); };
  double ip = 1.0, iq = 0.0;
  if (minus) {
    double sp = 0.0, sq = 0.0;
    for (int j = w0 + lane; j < w1; j += 32) { sp += ep(j); sq += eq(j); }
    sp = block_sum(sp, red);
    sq = block_sum(sq, red);
    if (tid == 0) { cta[0] = sp; cta[1] = sq; }
    cluster.sync();
    sp = sq = 0.0;
    for (int k = 0; k < C; ++k) {
      const double* o = cluster.map_shared_rank(cta, k);
      sp += o[0];
      sq += o[1];
    }
    ip = 1.0 / sp;
    iq = 1.0 / sq;
  }
  int plain = without >= 0 || minus ? 0 : 1; // 1: w = p
  for (;;) {
    auto weight = [&](int j) {
      const double e = ep(j);
      if (plain) return e;
      if (minus) return fmax(__dsub_rn(__dmul_rn(e, ip), __dmul_rn(eq(j), iq)), 0.0);   // 0 where the two are equal
      return j == without ? 0.0 : e;
    };
    double mine = 0.0;
    for (int j = w0 + lane; j < w1; j += 32) mine += weight(j);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, off);
    if (lane == 0) of_warp[warp] = mine;
    __syncthreads();
    if (tid == 0) {
      double v = 0.0;
      for (int w = 0; w < kWarps; ++w) v += of_warp[w];
      cta[2 + plain] = v;
    }
    cluster.sync();
    double total = 0.0;
    for (int k = 0; k < C; ++k) total += *cluster.map_shared_rank(cta + 2 + plain, k);
    if (!(total > 0.0) && !plain) { plain = 1; continue; }             // p <= q everywhere: the target itself
    const double goal = (double)p.sample_u[b] * total;
    // the first part whose running sum passes the goal; by rounding there may be none, then the last with any weight
    double run = 0.0, before = 0.0;
    int at = 0;
    for (int k = 0; k < C; ++k) {
      const double v = *cluster.map_shared_rank(cta + 2 + plain, k);
      if (v > 0.0) { at = k; before = run; if (run + v > goal) break; }
      run += v;
    }
    if (at == rank) {
      int aw = 0;
      run = before;
      for (int w = 0; w < kWarps; ++w) {
        const double v = of_warp[w];
        if (v > 0.0) { aw = w; before = run; if (run + v > goal) break; }
        run += v;
      }
      if (aw == warp) {                      // lanes take neighbouring runs of the warp's tokens
        const int per = (w1 - w0 + 31) / 32, l0 = min(w1, w0 + lane * per), l1 = min(w1, l0 + per);
        double v = 0.0;
        for (int j = l0; j < l1; ++j) v += weight(j);
        double incl = v;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const double u = __shfl_up_sync(0xffffffffu, incl, off);
          if (lane >= off) incl += u;
        }
        const unsigned passes = __ballot_sync(0xffffffffu, v > 0.0 && before + incl > goal), some = __ballot_sync(0xffffffffu, v > 0.0);
        const int who = passes ? __ffs(passes) - 1 : 31 - __clz(some);
        if (lane == who) {
          double sum = before + incl - v;
          int chosen = l0;
          for (int j = l0; j < l1; ++j) {
            const double wj = weight(j);
            sum += wj;
            if (wj > 0.0) { chosen = j; if (sum > goal) break; }
          }
          p.tokens_out[stop] = chosen;
        }
      }
    }
    break;
  }
  cluster.sync();                            // no CTA leaves while others read its sums
}

template <typename T>
int32_t launch_verify(Ctx* ctx, const VerifyParams& p) {
  LMB_CUDA(launch_k_opt(false, statistics_kernel<T>, dim3((unsigned)p.splits, (unsigned)p.rows), dim3(kStatThreads), 0, ctx->stream, p));
  ctx->launches++;
  const int C = p.vocab <= 4096 ? 1 : 8;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.n_seq * C));
  cfg.blockDim = dim3(kChooseThreads);
  cfg.stream = ctx->stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  LMB_CUDA(cudaLaunchKernelEx(&cfg, choose_kernel<T>, p));
  ctx->launches++;
  return LMB200_OK;
}

}  // namespace
}  // namespace lmb

using namespace lmb;

extern "C" int32_t lmb200_verify_drafts_workspace(int32_t rows, int64_t* bytes) {
  LMB_REQUIRE(bytes && rows >= 0, "verify_drafts_workspace: bad argument");
  *bytes = std::max<int64_t>(16, (int64_t)rows * kSplits * (int64_t)sizeof(float4));
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
  LMB_CUDA(cudaSetDevice(ctx->device));
  if (rows == 0) {
    LMB_CUDA(cudaMemsetAsync(n_out, 0, (size_t)n_seq * 4, ctx->stream));
    LMB_CUDA(cudaMemsetAsync(drop, 0, (size_t)n_seq * 4, ctx->stream));
    return LMB200_OK;
  }
  VerifyParams p = {target, draft, target_stride, draft_stride, vocab, rows, n_seq, vocab <= 4096 ? 1 : kSplits, cu_rows, tokens, temperature, accept_u, sample_u,
                    tokens_out, n_out, drop, ctx->dev_err, static_cast<float4*>(workspace)};
  return dtype == LMB200_F32 ? launch_verify<float>(ctx, p) : launch_verify<__nv_bfloat16>(ctx, p);
}
