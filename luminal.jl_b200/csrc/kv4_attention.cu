// Attention over the 4-bit paged cache (lmb200_kv4_attention).
#include <math_constants.h>

#include "kv4.cuh"
#include "pdl.cuh"

namespace lmb {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kThreads = 128;

struct Kv4Params {
  const void* q;
  void* out;
  int64_t q_stride, out_stride;
  int rows, n_seq, max_pages, n_pages, shift, heads, G, D, window;
  float scale;
  const int *cu_rows, *lens, *table;
  const uint8_t* pages;
  int* dev_err;
};

// One CTA per row and query head, its threads over keys for the scores and over features for the values.
template <typename T>
__global__ void __launch_bounds__(kThreads) kv4_attention_kernel(const Kv4Params p) {
  __shared__ float q[256], w[kThreads], red[8];
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.x, hq = blockIdx.y, h = hq / p.G, tid = threadIdx.x, D = p.D, NG = kv4::groups(D);
  if (r == 0 && hq == 0)                     // one CTA looks the offsets and lengths over
    for (int b = tid; b < p.n_seq; b += kThreads)
      if (p.cu_rows[b] < 0 || p.cu_rows[b + 1] < p.cu_rows[b] || p.cu_rows[b + 1] > p.rows || p.lens[b] < 0 || p.lens[b] > p.max_pages << p.shift)
        atomicExch(p.dev_err, kv4::kErrPage);
  int lo = 0, hi = p.n_seq;
  while (lo < hi) {                          // the first sequence that ends behind row r
    const int mid = (lo + hi) >> 1;
    if (p.cu_rows[mid + 1] <= r) lo = mid + 1; else hi = mid;
  }
  if (lo >= p.n_seq || r < p.cu_rows[lo]) return;
  const int b = lo, size1 = (1 << p.shift) - 1;
  const int len = min(max(p.lens[b], 0), p.max_pages << p.shift);
  const int position = len - (p.cu_rows[b + 1] - r);
  const int from = p.window > 0 ? max(0, position - p.window + 1) : 0;
  const T* qr = reinterpret_cast<const T*>(p.q) + r * p.q_stride + hq * D;
  for (int d = tid; d < D; d += kThreads) q[d] = to_f32(qr[d]) * p.scale * kLog2e;
  float M = -CUDART_INF_F, l = 0.f, o0 = 0.f, o1 = 0.f;
  for (int k0 = from; k0 <= position; k0 += kThreads) {
    __syncthreads();
    const int key = k0 + tid;
    float s = -CUDART_INF_F;
    const int n = min(kThreads, position + 1 - k0);
    if (tid < n) {
      const int page = p.table[(int64_t)b * p.max_pages + (key >> p.shift)];
      if ((unsigned)page < (unsigned)p.n_pages) {
        const uint8_t* block = p.pages + (((int64_t)page * p.heads + h) * (1 << (p.shift - 4)) + ((key & size1) >> 4)) * kv4::block_bytes(D);
        const __half* meta = reinterpret_cast<const __half*>(block + 16 * D);
        s = 0.f;
        for (int d = 0; d < D; ++d) {
          const int n4 = block[kv4::key_byte(key & 15, d)] >> ((d & 8) ? 4 : 0) & 15, at = kv4::key_meta(key & 15, d >> 5);
          s = fmaf(q[d], fmaf((float)n4, __half2float(meta[at]), __half2float(meta[D / 2 + at])), s);
        }
      } else {
        atomicExch(p.dev_err, kv4::kErrPage);
      }
    }
    float top = s;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    if ((tid & 31) == 0) red[tid >> 5] = top;
    __syncthreads();
    const float Mn = fmaxf(M, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]))), Mu = Mn == -CUDART_INF_F ? 0.f : Mn;
    const float fade = exp2f(M - Mu), e = exp2f(s - Mu);
    w[tid] = e;
    float sum = e;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if ((tid & 31) == 0) red[4 + (tid >> 5)] = sum;
    __syncthreads();
    l = l * fade + ((red[4] + red[5]) + (red[6] + red[7]));
    M = Mn;
    for (int i = 0, d = tid; d < D; ++i, d += kThreads) {
      float o = (i ? o1 : o0) * fade;
      for (int j = 0; j < n; ++j) {
        if (w[j] == 0.f) continue;           // also keys of a page that is not there
        const int kk = k0 + j;
        const int page = p.table[(int64_t)b * p.max_pages + (kk >> p.shift)];
        const uint8_t* block = p.pages + (((int64_t)page * p.heads + h) * (1 << (p.shift - 4)) + ((kk & size1) >> 4)) * kv4::block_bytes(D);
        const __half* meta = reinterpret_cast<const __half*>(block + 16 * D) + D;
        const int n4 = block[8 * D + kv4::value_byte(kk & 15, d)] >> ((d & 8) ? 4 : 0) & 15, at = kv4::value_meta(kk & 15, d >> 5);
        o = fmaf(w[j], fmaf((float)n4, __half2float(meta[at]), __half2float(meta[D / 2 + at])), o);
      }
      if (i) o1 = o; else o0 = o;
    }
  }
  T* out = reinterpret_cast<T*>(p.out) + r * p.out_stride + hq * D;
  for (int i = 0, d = tid; d < D; ++i, d += kThreads) out[d] = from_f32<T>(l > 0.f || l != l ? (i ? o1 : o0) / l : 0.f);
}

}  // namespace
}  // namespace lmb

using namespace lmb;

extern "C" int32_t lmb200_kv4_attention_workspace(lmb200_ctx h, int32_t head_dim, int64_t* bytes) {
  Ctx* ctx = ctx_from(h);
  if (!ctx) return LMB200_EINVAL;
  LMB_REQUIRE(bytes, "kv4_attention_workspace: null argument");
  LMB_TRY(kv4::check_cache("kv4_attention_workspace", 1, head_dim, 1, 16));
  *bytes = 16;
  return LMB200_OK;
}

extern "C" int32_t lmb200_kv4_attention(lmb200_ctx h, int32_t dtype, const void* q, int64_t q_stride, void* out, int64_t out_stride, int32_t rows, int32_t n_seq,
                                        const int32_t* cu_rows, const int32_t* lens, const int32_t* table, int32_t max_pages, const void* pages, int32_t n_pages,
                                        int32_t page_size, int32_t n_kv_heads, int32_t group, int32_t head_dim, float scale, int32_t window, void* workspace,
                                        int64_t workspace_bytes) {
  Ctx* ctx = ctx_from(h);
  if (!ctx) return LMB200_EINVAL;
  LMB_REQUIRE(dtype == LMB200_F32 || dtype == LMB200_BF16, "kv4_attention: dtype %d", dtype);
  LMB_TRY(kv4::check_cache("kv4_attention", n_kv_heads, head_dim, n_pages, page_size));
  LMB_REQUIRE(group >= 1 && (int64_t)n_kv_heads * group <= 65535, "kv4_attention: %d query heads for each of %d kv heads", group, n_kv_heads);
  LMB_REQUIRE(rows >= 0 && n_seq >= 1 && n_seq <= 8192 && window >= 0, "kv4_attention: %d rows, %d sequences (1 to 8192), window %d", rows, n_seq, window);
  LMB_REQUIRE(max_pages >= 1 && (int64_t)max_pages * page_size <= INT32_MAX, "kv4_attention: block tables of %d pages", max_pages);
  LMB_REQUIRE(rows == 0 || (q && out && cu_rows && lens && table && pages && workspace), "kv4_attention: null pointer");
  const int64_t width = (int64_t)n_kv_heads * group * head_dim;
  LMB_REQUIRE(q_stride >= width && out_stride >= width, "kv4_attention: row strides %lld and %lld for rows of %lld elements", (long long)q_stride, (long long)out_stride,
              (long long)width);
  const int vec = dtype == LMB200_F32 ? 4 : 8;
  LMB_REQUIRE(q_stride % vec == 0 && out_stride % vec == 0 && (uintptr_t)q % 16 == 0 && (uintptr_t)out % 16 == 0 && (uintptr_t)pages % 16 == 0 &&
                  (uintptr_t)workspace % 16 == 0, "kv4_attention: rows, pages and workspace must start on 16-byte boundaries");
  int64_t need = 0;
  LMB_TRY(lmb200_kv4_attention_workspace(h, head_dim, &need));
  LMB_REQUIRE(workspace_bytes >= need, "kv4_attention: a workspace of %lld bytes, %lld are needed", (long long)workspace_bytes, (long long)need);
  if (rows == 0) return LMB200_OK;
  LMB_CUDA(cudaSetDevice(ctx->device));
  Kv4Params p = {q, out, q_stride, out_stride, rows, n_seq, max_pages, n_pages, kv4::page_shift(page_size), n_kv_heads, group, head_dim, window,
                 scale, cu_rows, lens, table, static_cast<const uint8_t*>(pages), ctx->dev_err};
  const dim3 grid((unsigned)rows, (unsigned)(n_kv_heads * group));
  if (dtype == LMB200_F32) LMB_CUDA(launch_k_opt(false, kv4_attention_kernel<float>, grid, dim3(kThreads), 0, ctx->stream, p));
  else LMB_CUDA(launch_k_opt(false, kv4_attention_kernel<__nv_bfloat16>, grid, dim3(kThreads), 0, ctx->stream, p));
  ctx->launches++;
  return LMB200_OK;
}
