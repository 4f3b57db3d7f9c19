// Attention over the 4-bit paged cache, bf16 queries: the instantiations.
#include "kv4_attention.cuh"

namespace lmb {
namespace kv4 {
namespace {
Variant g_variants[9][5];
}
const Variant* variant_bf16(int NG, int NT) { return &g_variants[NG][NT]; }

int32_t configure_bf16() {
#define KV4_ONE(NG, NT) LMB_TRY((configure_one<__nv_bfloat16, NG, NT>(&g_variants[NG][NT])))
#define KV4_NARROW(NG) KV4_ONE(NG, 1); KV4_ONE(NG, 2); KV4_ONE(NG, 3); KV4_ONE(NG, 4)
#define KV4_WIDE(NG) KV4_ONE(NG, 1); KV4_ONE(NG, 2)
  KV4_NARROW(1); KV4_NARROW(2); KV4_NARROW(3); KV4_NARROW(4);
  KV4_WIDE(5); KV4_WIDE(6); KV4_WIDE(7); KV4_WIDE(8);
  return LMB200_OK;
}

}  // namespace kv4
}  // namespace lmb
