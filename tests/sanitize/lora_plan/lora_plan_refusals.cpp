// lora_plan_refusals.cpp -- imq_qmm_lora_plan and the factors by rank of imq_lora.h in a
// host-only sanitized build (TEST INFRASTRUCTURE ONLY; no GPU).
//
// Prints "lora_plan_refusals: <n> checks"; any wrong status or plan ends it.
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "ctx.hpp"
#include "imq.h"
#include "imq_lora.h"
#include "lora.hpp"

namespace imq {
LoraPlan next;  // what the planner says
bool by_rows, join_few;
hipError_t launch_lora_shrink(const LoraArgs&, const void*, int, int, int, hipStream_t) {
  return hipErrorNoDevice;
}
hipError_t launch_lora_join(const LoraArgs&, const float*, int, void*, int, int, int, hipStream_t) {
  return hipErrorNoDevice;
}
hipError_t launch_lora_order(const LoraArgs&, int32_t*, int32_t*, int, hipStream_t) { return hipErrorNoDevice; }
LoraPlan lora_plan(int, int, int, int, int, int) { return next; }
bool lora_by_rows(int, int, bool, int, int) { return by_rows; }
bool lora_join_few(int, int, int, int) { return join_few; }
hipError_t launch_qgemm_lora(const LoraPlan&, const uint32_t*, const void*, const void*, const void*,
                             const LoraArgs&, float*, void*, int, int, int, int, hipStream_t) {
  return hipErrorNoDevice;
}
}  // namespace imq

namespace {

int checks = 0;
imq_ctx ctx;
alignas(16) char mem[4096];

void need(bool ok, const char* what) {
  ++checks;
  if (ok) return;
  fprintf(stderr, "lora_plan_refusals: %s (%s)\n", what, imq_last_error(&ctx));
  exit(4);
}

imq_lora set() {
  return imq_lora{mem, mem + 1024, reinterpret_cast<int32_t*>(mem), reinterpret_cast<float*>(mem), 3, 64, 32, 0};
}

void plan(const char* what, imq::LoraPlan p, bool by_rows, bool join_few, int kernel, int tile_rows, int splits, int u_rows,
          int grouped, int join_tiles) {
  imq::next = p, imq::by_rows = by_rows, imq::join_few = join_few;
  const imq_lora l = set();
  imq_lora_plan_info i;
  size_t bytes = 0;
  need(imq_qmm_lora_plan(&ctx, &l, 128, 96, 70, IMQ_BF16, &i) == IMQ_OK, what);
  need(imq_qmm_lora_workspace(&ctx, &l, 128, 96, 70, IMQ_BF16, &bytes) == IMQ_OK && bytes == i.workspace_bytes, what);
  need(i.kernel == kernel && i.tile_rows == tile_rows && i.splits == splits && i.u_rows == u_rows && i.grouped == grouped &&
           i.join_tiles == join_tiles, what);
}

}  // namespace

int main() {
  ctx.device = 1 << 20;
  plan("few rows", imq::LoraPlan{1, 5, 0, 0, 0, false, 100}, false, true, IMQ_LORA_FEW, 0, 5, 1, 0, 0);
  plan("split, tiles", imq::LoraPlan{0, 4, 2, 1, 3, false, 100}, false, false, IMQ_LORA_SPLIT, 64, 4, 0, 0, 1);
  plan("all of K, rows", imq::LoraPlan{0, 1, 8, 2, 3, false, 100}, true, true, IMQ_LORA_SPLIT, 256, 1, 1, 0, 0);
  plan("tiles", imq::LoraPlan{0, 0, 6, 2, 3, true, 0}, false, true, IMQ_LORA_TILES, 192, 1, 0, 1, 0);
  plan("register-staged", imq::LoraPlan{}, true, false, IMQ_LORA_TILES_REG, 0, 1, 1, 0, 0);
  imq_lora l = set();
  imq_lora_plan_info i;
  size_t bytes;
  need(imq_qmm_lora_plan(nullptr, &l, 128, 96, 5, IMQ_BF16, &i) == IMQ_EINVAL, "null context");
  need(imq_qmm_lora_plan(&ctx, nullptr, 128, 96, 5, IMQ_BF16, &i) == IMQ_EINVAL, "null adapters");
  need(imq_qmm_lora_plan(&ctx, &l, 128, 96, 5, IMQ_BF16, nullptr) == IMQ_EINVAL, "null output");
  need(imq_qmm_lora_plan(&ctx, &l, 128, 96, 5, IMQ_F32, &i) == IMQ_EUNSUPPORTED, "f32");
  for (int bad : {0, -1, INT32_MIN}) {
    need(imq_qmm_lora_plan(&ctx, &l, bad, 96, 5, IMQ_BF16, &i) == IMQ_EINVAL, "k");
    need(imq_qmm_lora_plan(&ctx, &l, 128, bad, 5, IMQ_BF16, &i) == IMQ_EINVAL, "n");
    need(imq_qmm_lora_plan(&ctx, &l, 128, 96, bad, IMQ_BF16, &i) == IMQ_EINVAL, "m");
  }
  for (int bad : {-1, 2, INT32_MIN, INT32_MAX}) {
    l.rank_scales = bad;
    need(imq_qmm_lora_workspace(&ctx, &l, 128, 96, 5, IMQ_F16, &bytes) == IMQ_EINVAL && strstr(imq_last_error(&ctx), "rank_scales"),
         "rank_scales");
    need(imq_qmm_lora_plan(&ctx, &l, 128, 96, 5, IMQ_F16, &i) == IMQ_EINVAL, "rank_scales of a plan");
    need(imq_qmm_lora(&ctx, reinterpret_cast<uint32_t*>(mem), mem, mem, mem, &l, reinterpret_cast<int32_t*>(mem), mem + 2048, 128, 96, 5,
                      64, 4, IMQ_F16, mem, 1 << 20, nullptr) == IMQ_EINVAL, "rank_scales of a call");
  }
  l.rank_scales = 1;
  need(imq_qmm_lora_workspace(&ctx, &l, 128, 96, 5, IMQ_F16, &bytes) == IMQ_OK, "factors by rank");
  printf("lora_plan_refusals: %d checks\n", checks);
  return 0;
}
