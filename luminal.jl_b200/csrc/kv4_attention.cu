// Attention over the 4-bit paged cache (lmb200_kv4_attention): the choice of a variant and its launch.
#include <algorithm>

#include "kv4_attention.cuh"

namespace lmb {
namespace {

// The grid of a variant: every CTA that fits on the GPU.  CTAs do not wait for one another, so fewer may run at a time.
int grid_of(const Ctx* ctx, const kv4::Variant* v) { return std::min(ctx->sm_count * std::max(1, v->ctas_per_sm), kv4::kMostShares); }

int64_t workspace_bytes_of(const Ctx* ctx, int D) {
  int64_t most = 0;
  for (int f32 = 0; f32 < 2; ++f32)
    for (int nt = 1; nt <= kv4::kMostTiles; ++nt)
      most = std::max<int64_t>(most, (int64_t)grid_of(ctx, f32 ? kv4::variant_f32(kv4::groups(D), nt) : kv4::variant_bf16(kv4::groups(D), nt)) * 2 * (8 * nt) * (D + 2) * 4);
  return kv4::kCounters * 4 + most;
}

}  // namespace

int32_t kv4_attention_configure() {
  LMB_TRY(kv4::configure_bf16());
  return kv4::configure_f32();
}

}  // namespace lmb

using namespace lmb;

extern "C" int32_t lmb200_kv4_attention_workspace(lmb200_ctx h, int32_t head_dim, int64_t* bytes) {
  Ctx* ctx = ctx_from(h);
  if (!ctx) return LMB200_EINVAL;
  LMB_REQUIRE(bytes, "kv4_attention_workspace: null argument");
  LMB_TRY(kv4::check_cache("kv4_attention_workspace", 1, head_dim, 1, 16));
  *bytes = workspace_bytes_of(ctx, head_dim);
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
  const int64_t capacity = (int64_t)max_pages * page_size;
  LMB_REQUIRE(max_pages >= 1 && capacity <= kv4::kMostTokens, "kv4_attention: block tables of %d pages (up to 2^30 tokens)", max_pages);
  LMB_REQUIRE(rows <= kv4::kMostTokens && (int64_t)rows * group <= INT32_MAX - 8 * kv4::kMostTiles, "kv4_attention: %d rows for each of %d heads", rows, group);     // rounded up to tiles in 32 bits
  LMB_REQUIRE(rows == 0 || (q && out && cu_rows && lens && table && pages && workspace), "kv4_attention: null pointer");
  const int64_t width = (int64_t)n_kv_heads * group * head_dim;
  LMB_REQUIRE(q_stride >= width && out_stride >= width, "kv4_attention: row strides %lld and %lld for rows of %lld elements", (long long)q_stride, (long long)out_stride,
              (long long)width);
  const int vec = dtype == LMB200_F32 ? 4 : 8;
  LMB_REQUIRE(q_stride % vec == 0 && out_stride % vec == 0 && (uintptr_t)q % 16 == 0 && (uintptr_t)out % 16 == 0 && (uintptr_t)pages % 16 == 0 &&
                  (uintptr_t)workspace % 16 == 0, "kv4_attention: rows, pages and workspace must start on 16-byte boundaries");
  const int64_t size = dtype == LMB200_F32 ? 4 : 2;
  LMB_REQUIRE(rows == 0 || (out == q && (out_stride == q_stride || rows == 1)) || kv4::apart(q, q_stride * size, out, out_stride * size, rows, width * size),
              "kv4_attention: out lies over q in part: it may be q with q's stride, or share no byte with it");
  const int64_t need = workspace_bytes_of(ctx, head_dim);
  LMB_REQUIRE(workspace_bytes >= need, "kv4_attention: a workspace of %lld bytes, %lld are needed", (long long)workspace_bytes, (long long)need);
  if (rows == 0) return LMB200_OK;
  // Query rows of one kv head that share a pass over its keys: 8, or 16 where that makes 3/5 as many passes or fewer (a pass for 16 takes 5/3 of one for 8).  Only the device knows
  // how many rows each sequence has; the average decides.  24 rows (6 drafts of 4 heads): 66 us as three eights, 74 as two sixteens; 16 rows: 44 and 42; 1024: 345 and 268.  Tiles of 24
  // and 32 rows leave registers for two CTAs an SM and were slower everywhere (71 and 92 us for the 24 rows).
  const bool f32 = dtype == LMB200_F32;
  const int NG = kv4::groups(head_dim);
  const int64_t each = ceil_div(rows, n_seq) * group;
  const int NT = ceil_div(each, 16) * 5 <= ceil_div(each, 8) * 3 ? 2 : 1;
  const kv4::Variant* v = f32 ? kv4::variant_f32(NG, NT) : kv4::variant_bf16(NG, NT);
  // units of work are counted in 32 bits
  const int64_t tiles = ceil_div((int64_t)rows * group, 8 * NT) + std::min(n_seq, rows), units = ceil_div(capacity, kv4::kUnit) + 1;
  LMB_REQUIRE(tiles * n_kv_heads <= UINT32_MAX / units, "kv4_attention: %d rows of %d heads over %d pages are too many for one call", rows, n_kv_heads * group, max_pages);
  LMB_CUDA(cudaSetDevice(ctx->device));
  const int grid = (int)std::min<int64_t>(grid_of(ctx, v), tiles * n_kv_heads * units);
  kv4::Params p = {};
  p.q = q; p.out = out; p.q_stride = q_stride; p.out_stride = out_stride;
  p.rows = rows; p.n_seq = n_seq; p.max_pages = max_pages; p.n_pages = n_pages; p.shift = kv4::page_shift(page_size);
  p.heads = n_kv_heads; p.G = group; p.window = window < capacity ? window : 0;
  p.scale = scale * 1.4426950408889634f;
  p.cu_rows = cu_rows; p.lens = lens; p.table = table;
  p.pages = static_cast<const uint8_t*>(pages);
  p.dev_err = ctx->dev_err;
  p.dev_arg = ctx->dev_arg;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.counters = reinterpret_cast<unsigned*>(ws);
  p.part_o = reinterpret_cast<float*>(ws + kv4::kCounters * 4);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + (int64_t)grid * 2 * 8 * NT * head_dim);
  LMB_CUDA(launch_k_opt(false, v->kernel, dim3((unsigned)grid), dim3(kv4::kThreads), (size_t)v->smem + kv4::seq_bytes(n_seq), ctx->stream, p));
  ctx->launches++;
  return LMB200_OK;
}
