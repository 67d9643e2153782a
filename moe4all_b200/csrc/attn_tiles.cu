#include "attn.cuh"
namespace infr {
int32_t launch_attn_tiles(infr_cuda_ctx* ctx, AttnParams p, const __half* k) {
  if (p.g > 16) return fail(ctx, INFR_CUDA_ERR_UNSUPPORTED, "attention: more than 16 query heads to a kv head");
  return launch_attn_rows(ctx, p, k, 16);
}
}  // namespace infr
