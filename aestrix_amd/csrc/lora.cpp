// lora.cpp -- the C entry points of include/imq_lora.h: argument checks, the workspace
// and the launches.
#include "ctx.hpp"
#include "imq_lora.h"
#include "lora.hpp"

using namespace imq::detail;

int imq::detail::check_lora(imq_ctx* ctx, const char* fn, const imq_lora* l, int k, int n, int m,
                            imq_dtype dtype) {
  if (!ctx) return fail(nullptr, IMQ_EINVAL, "%s: null context", fn);
  if (!l) return fail(ctx, IMQ_EINVAL, "%s: null adapters", fn);
  if (dtype != IMQ_BF16 && dtype != IMQ_F16)
    return fail(ctx, IMQ_EUNSUPPORTED, "%s: dtype %d (bf16 and f16 are provided)", fn, (int)dtype);
  if (k <= 0 || n <= 0 || m <= 0 || k % 64 != 0)
    return fail(ctx, IMQ_EINVAL, "%s: shape K=%d N=%d M=%d (K a multiple of 64, all > 0)", fn, k, n, m);
  // 32 rows of x or A are addressed with 32-bit byte offsets.
  if (k > 1 << 25) return fail(ctx, IMQ_EUNSUPPORTED, "%s: K=%d (up to 2^25)", fn, k);
  if (l->count <= 0 || l->rows < 0 || l->rows % 16 != 0)
    return fail(ctx, IMQ_EINVAL, "%s: %d adapters of %d rows (whole 16s)", fn, l->count, l->rows);
  if (l->max_rank <= 0 || l->max_rank % 16 != 0)
    return fail(ctx, IMQ_EINVAL, "%s: largest rank %d (a multiple of 16)", fn, l->max_rank);
  if (l->max_rank > imq::kLoraMaxRank)
    return fail(ctx, IMQ_EUNSUPPORTED, "%s: rank %d (up to %d are provided)", fn, l->max_rank,
                imq::kLoraMaxRank);
  if (l->rank_scales != 0 && l->rank_scales != 1)
    return fail(ctx, IMQ_EINVAL, "%s: rank_scales %d (0 or 1)", fn, l->rank_scales);
  if (!l->a || !l->b || !l->first || !l->scale)
    return fail(ctx, IMQ_EINVAL, "%s: null device pointer (a=%p b=%p first=%p scale=%p)", fn, l->a, l->b,
                (const void*)l->first, (const void*)l->scale);
  if (!aligned(l->a, 16) || !aligned(l->b, 16) || !aligned(l->first, 4) || !aligned(l->scale, 4))
    return fail(ctx, IMQ_EINVAL, "%s: a and b must be 16-byte, first and scale 4-byte aligned", fn);
  return IMQ_OK;
}

namespace {

// u, then the partial sums or the order and the adapters of the places.
size_t workspace(const imq_lora* l, const imq::LoraPlan& p, int m) {
  return imq::lora_u_bytes(m, l->max_rank) + (p.order ? (size_t)m * 8 : p.bytes);
}

}  // namespace

extern "C" {

int imq_qmm_lora_workspace(imq_ctx* ctx, const imq_lora* lora, int k, int n, int m, imq_dtype dtype,
                           size_t* bytes) {
  const char* fn = "imq_qmm_lora_workspace";
  const int rc = check_lora(ctx, fn, lora, k, n, m, dtype);
  if (rc != IMQ_OK) return rc;
  if (!bytes) return fail(ctx, IMQ_EINVAL, "%s: null output", fn);
  *bytes = workspace(lora, imq::lora_plan(k, n, m, lora->count, lora->max_rank, (int)dtype), m);
  return IMQ_OK;
}

int imq_qmm_lora(imq_ctx* ctx, const uint32_t* w, const void* scales, const void* biases,
                 const void* x, const imq_lora* lora, const int32_t* which, void* y, int k, int n,
                 int m, int group_size, int bits, imq_dtype dtype, void* ws, size_t ws_bytes,
                 imq_stream stream) {
  const char* fn = "imq_qmm_lora";
  int rc = check_qmm(ctx, fn, w, scales, biases, x, y, k, n, m, group_size, bits, dtype);
  if (rc != IMQ_OK || (rc = check_lora(ctx, fn, lora, k, n, m, dtype)) != IMQ_OK) return rc;
  if (!which || !aligned(which, 4))
    return fail(ctx, IMQ_EINVAL, "%s: which=%p must be a 4-byte aligned device pointer", fn,
                (const void*)which);
  const imq::LoraPlan plan = imq::lora_plan(k, n, m, lora->count, lora->max_rank, (int)dtype);
  const size_t need = workspace(lora, plan, m);
  if (!ws || !aligned(ws, 16) || ws_bytes < need)
    return fail(ctx, IMQ_EINVAL, "%s: workspace %p of %zu bytes (16-byte aligned, %zu are needed)", fn, ws,
                ws_bytes, need);
  if (x == y) return fail(ctx, IMQ_EINVAL, "%s: y is x", fn);
  if ((rc = bind_device(ctx)) != IMQ_OK) return rc;
  imq::LoraArgs l{static_cast<const uint16_t*>(lora->a), static_cast<const uint16_t*>(lora->b),
                        lora->first, lora->scale, which, static_cast<uint16_t*>(ws),
                        lora->count, lora->rows, lora->max_rank, lora->rank_scales, nullptr};
  char* rest = static_cast<char*>(ws) + imq::lora_u_bytes(m, lora->max_rank);
  auto* part = reinterpret_cast<float*>(rest);
  const auto st = static_cast<hipStream_t>(stream);
  hipError_t e = hipSuccess;
  if (plan.order) {
    auto* order = reinterpret_cast<int32_t*>(rest);
    e = imq::launch_lora_order(l, order, order + m, m, st);
    l.order = order, l.which = order + m;
  }
  if (e == hipSuccess && !plan.few) e = imq::launch_lora_shrink(l, x, k, m, (int)dtype, st);
  if (e == hipSuccess)
    e = imq::launch_qgemm_lora(plan, w, scales, biases, x, l, part, y, k, n, m, (int)dtype, st);
  if (e == hipSuccess && plan.splits > 0)
    e = imq::launch_lora_join(l, part, plan.splits, y, n, m, (int)dtype, st);
  return e == hipSuccess ? IMQ_OK : hip_fail(ctx, e, fn);
}

}  // extern "C"
