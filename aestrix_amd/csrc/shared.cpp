// shared.cpp -- the C entry point of attention behind shared keys
// (imq_attention_shared, include/imq_core.h): argument checks and the launch.
#include "core_checks.hpp"
#include "core_kernels.hpp"
#include "ctx.hpp"
#include "imq_core.h"

using namespace imq::detail;

namespace {

// The shared keys of a call whose other arguments are checked.
int check_shared(imq_ctx* ctx, const char* fn, const imq_attention_args* p, const imq_shared_keys* k,
                 imq::AttnShared* sh) {
  if (!k) return fail(ctx, IMQ_EINVAL, "%s: null shared keys", fn);
  if (k->rows < 0) return fail(ctx, IMQ_EINVAL, "%s: %d shared keys", fn, k->rows);
  if ((int64_t)k->rows + p->max_k >= (int64_t)1 << 31)
    return fail(ctx, IMQ_EINVAL, "%s: %d shared and %d own keys", fn, k->rows, p->max_k);
  if (reach({{k->rows, k->k_row}, {p->kv_heads, k->k_head}}) < 0 ||
      reach({{k->rows, k->v_row}, {p->kv_heads, k->v_head}}) < 0)
    return fail(ctx, IMQ_EINVAL, "%s: a negative stride of the shared keys, or 2^60 elements", fn);
  if (k->rows > 0 && p->n_seq > 0 && p->max_q > 0) {
    if (!k->k || !k->v)
      return fail(ctx, IMQ_EINVAL, "%s: null device pointer (shared k=%p v=%p)", fn, k->k, k->v);
    if (p->out == k->k || p->out == k->v)
      return fail(ctx, IMQ_EINVAL, "%s: out is the shared k or v", fn);
    if (!aligned(k->k, 2) || !aligned(k->v, 2))
      return fail(ctx, IMQ_EINVAL, "%s: shared k and v must be 2-byte aligned", fn);
  }
  *sh = imq::AttnShared{k->k, k->v, k->k_row, k->k_head, k->v_row, k->v_head, k->rows};
  return IMQ_OK;
}

}  // namespace

extern "C" {

int imq_attention_shared(imq_ctx* ctx, const imq_attention_args* args,
                         const imq_shared_keys* shared, imq_stream stream) {
  const char* fn = "imq_attention_shared";
  imq::AttnArgs a{};
  imq::AttnShared sh{};
  int rc = check_attention(ctx, fn, args, &a);
  if (rc != IMQ_OK || (rc = check_shared(ctx, fn, args, shared, &sh)) != IMQ_OK) return rc;
  if (sh.rows == 0) return imq_attention(ctx, args, stream);
  if (a.n_seq == 0 || a.max_q == 0) return IMQ_OK;
  if ((rc = bind_device(ctx)) != IMQ_OK) return rc;
  const auto st = static_cast<hipStream_t>(stream);
  imq::SharedPlan plan = imq::attention_shared_plan(a, sh, ctx->cus, true);
  SplitHold hold;  // until the join is enqueued
  if (plan.bytes > 0) {
    hold = split_ws(ctx, st, plan.bytes);
    // It would have to grow under capture, or memory is short.
    if (!hold.ws.p) plan = imq::attention_shared_plan(a, sh, ctx->cus, false);
  }
  const hipError_t e = args->dtype == IMQ_BF16
                           ? imq::launch_attention_shared_bf16(a, sh, plan, hold.ws.p, st)
                           : imq::launch_attention_shared_f16(a, sh, plan, hold.ws.p, st);
  return e == hipSuccess ? IMQ_OK : hip_fail(ctx, e, fn);
}

int imq_attention_shared_plan(imq_ctx* ctx, const imq_attention_args* args, const imq_shared_keys* shared,
                              imq_shared_plan_info* out) {
  const char* fn = "imq_attention_shared_plan";
  imq::AttnArgs a{};
  imq::AttnShared sh{};
  int rc = check_attention(ctx, fn, args, &a);
  if (rc != IMQ_OK || (rc = check_shared(ctx, fn, args, shared, &sh)) != IMQ_OK) return rc;
  if (!out) return fail(ctx, IMQ_EINVAL, "%s: null output", fn);
  if (sh.rows == 0) {
    const imq::AttnPlan p = imq::attention_plan(a, ctx->cus);
    const bool few = p.kernel == IMQ_ATTENTION_FEW;
    out->kernel = few ? IMQ_SHARED_STREAM : p.kernel == IMQ_ATTENTION_TILES ? IMQ_SHARED_TILES : IMQ_SHARED_ROWS;
    out->tile_rows = p.tile_rows;
    out->splits = few ? 0 : p.splits;
    out->own_splits = few ? p.splits : 0;
    out->workspace_bytes = p.bytes;
    return IMQ_OK;
  }
  const imq::SharedPlan p = imq::attention_shared_plan(a, sh, ctx->cus, true);
  out->kernel = p.kernel;
  const bool apart = p.kernel == IMQ_SHARED_STREAM || p.kernel == IMQ_SHARED_PACKED;
  const bool tiles = p.kernel == IMQ_SHARED_TILES;
  out->tile_rows = apart ? p.s_rows : tiles ? p.tiles.tile_rows : 1;
  out->splits = apart ? p.s_splits : tiles ? p.tiles.splits : 1;
  out->own_splits = apart ? p.o_splits : 0;
  out->workspace_bytes = p.bytes;
  return IMQ_OK;
}

}  // extern "C"
