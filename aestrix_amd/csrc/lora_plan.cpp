// lora_plan.cpp -- what an imq_qmm_lora call runs (imq_qmm_lora_plan, include/imq_lora.h).
#include "lora.hpp"

using namespace imq::detail;

extern "C" int imq_qmm_lora_plan(imq_ctx* ctx, const imq_lora* lora, int k, int n, int m, imq_dtype dtype,
                                 imq_lora_plan_info* out) {
  const char* fn = "imq_qmm_lora_plan";
  int rc = check_lora(ctx, fn, lora, k, n, m, dtype);
  if (rc != IMQ_OK) return rc;
  if (!out) return fail(ctx, IMQ_EINVAL, "%s: null output", fn);
  const imq::LoraPlan p = imq::lora_plan(k, n, m, lora->count, lora->max_rank, (int)dtype);
  out->kernel = p.few ? IMQ_LORA_FEW : p.splits > 0 ? IMQ_LORA_SPLIT : p.mt > 0 ? IMQ_LORA_TILES : IMQ_LORA_TILES_REG;
  out->tile_rows = p.few ? 0 : 32 * p.mt;
  out->splits = p.splits > 0 ? p.splits : 1;
  out->u_rows = p.few || imq::lora_by_rows(lora->count, lora->max_rank, p.order, k, m);
  out->grouped = p.order;
  out->join_tiles = p.splits > 0 && !imq::lora_join_few(n, m, lora->count, lora->max_rank);
  return imq_qmm_lora_workspace(ctx, lora, k, n, m, dtype, &out->workspace_bytes);
}
