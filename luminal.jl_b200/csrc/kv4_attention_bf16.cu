// Attention over the 4-bit paged cache, bf16 queries: the instantiations.
#include "kv4_attention.cuh"

namespace lmb {
namespace kv4 {
namespace {
Variant g_variants[9][kMostTiles + 1];
}
const Variant* variant_bf16(int NG, int NT) { return &g_variants[NG][NT]; }

int32_t configure_bf16() {
#define KV4_BOTH(NG)                                            \
  LMB_TRY((configure_one<__nv_bfloat16, NG, 1>(&g_variants[NG][1]))); \
  LMB_TRY((configure_one<__nv_bfloat16, NG, 2>(&g_variants[NG][2])))
  KV4_BOTH(1); KV4_BOTH(2); KV4_BOTH(3); KV4_BOTH(4);
  KV4_BOTH(5); KV4_BOTH(6); KV4_BOTH(7); KV4_BOTH(8);
#undef KV4_BOTH
  return LMB200_OK;
}

}  // namespace kv4
}  // namespace lmb
