// lora_refusals.cpp -- the argument checks of imq_lora.h's entry points in a
// host-only sanitized build (TEST INFRASTRUCTURE ONLY; no GPU).
//
// Every call goes to a context of a device that does not exist: arguments that
// the checks let through fail at hipSetDevice (IMQ_EHIP), refused ones before
// that.  Prints "lora_refusals: <n> checks"; any wrong status ends it.
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "ctx.hpp"
#include "imq.h"
#include "imq_lora.h"
#include "lora.hpp"

namespace imq {
hipError_t launch_lora_shrink(const LoraArgs&, const void*, int, int, int, hipStream_t) {
  return hipErrorNoDevice;
}
hipError_t launch_lora_join(const LoraArgs&, const float*, int, void*, int, int, int, hipStream_t) {
  return hipErrorNoDevice;
}
hipError_t launch_lora_order(const LoraArgs&, int32_t*, int32_t*, int, hipStream_t) { return hipErrorNoDevice; }
LoraPlan lora_plan(int, int n, int m, int, int, int) { return LoraPlan{0, 2, 1, 2, 2, false, (size_t)8 * m * n}; }
hipError_t launch_qgemm_lora(const LoraPlan&, const uint32_t*, const void*, const void*, const void*,
                             const LoraArgs&, float*, void*, int, int, int, int, hipStream_t) {
  return hipErrorNoDevice;
}
}  // namespace imq

namespace {

int checks = 0;
imq_ctx ctx;
alignas(16) char mem[4096];

struct Call {
  imq_lora l{mem, mem + 1024, reinterpret_cast<int32_t*>(mem), reinterpret_cast<float*>(mem), 3, 64, 32};
  const uint32_t* w = reinterpret_cast<uint32_t*>(mem);
  const void *s = mem, *b = mem, *x = mem;
  const int32_t* which = reinterpret_cast<int32_t*>(mem);
  void *y = mem + 2048, *ws = mem;
  size_t bytes = (size_t)1 << 20;
  int k = 128, n = 96, m = 5, group = 64, bits = 4, dtype = IMQ_F16;
};

template <class F>
void lora(int want, const char* what, F change, int want_size = -1) {
  Call c;
  change(c);
  size_t need = 0;
  const int size = imq_qmm_lora_workspace(&ctx, &c.l, c.k, c.n, c.m, (imq_dtype)c.dtype, &need);
  const int got = imq_qmm_lora(&ctx, c.w, c.s, c.b, c.x, &c.l, c.which, c.y, c.k, c.n, c.m, c.group, c.bits,
                               (imq_dtype)c.dtype, c.ws, c.bytes, nullptr);
  checks += 2;
  if (got != want || strlen(imq_last_error(&ctx)) == 0 || (want_size >= 0 && size != want_size) ||
      (size == IMQ_OK) != (need >= 16)) {
    fprintf(stderr, "lora_refusals: %s returned %d, expected %d; the size's %d, %zu bytes (%s)\n", what, got,
            want, size, need, imq_last_error(&ctx));
    exit(4);
  }
}

}  // namespace

int main() {
  ctx.device = 1 << 20;
  lora(IMQ_EHIP, "good", [](Call&) {}, IMQ_OK);
  lora(IMQ_EHIP, "bf16", [](Call& c) { c.dtype = IMQ_BF16; }, IMQ_OK);
  lora(IMQ_EHIP, "rank 256", [](Call& c) { c.l.max_rank = 256; }, IMQ_OK);
  lora(IMQ_EHIP, "odd columns", [](Call& c) { c.n = 1; }, IMQ_OK);
  lora(IMQ_EUNSUPPORTED, "f32", [](Call& c) { c.dtype = IMQ_F32; }, IMQ_EUNSUPPORTED);
  lora(IMQ_EUNSUPPORTED, "no dtype", [](Call& c) { c.dtype = 3; }, IMQ_EUNSUPPORTED);
  lora(IMQ_EUNSUPPORTED, "rank 272", [](Call& c) { c.l.max_rank = 272; }, IMQ_EUNSUPPORTED);
  lora(IMQ_EUNSUPPORTED, "groups of 32", [](Call& c) { c.group = 32; });
  lora(IMQ_EUNSUPPORTED, "8 bits", [](Call& c) { c.bits = 8; });
  for (int bad : {0, -1, INT32_MIN}) {
    lora(IMQ_EINVAL, "k", [&](Call& c) { c.k = bad; }, IMQ_EINVAL);
    lora(IMQ_EINVAL, "n", [&](Call& c) { c.n = bad; }, IMQ_EINVAL);
    lora(IMQ_EINVAL, "m", [&](Call& c) { c.m = bad; }, IMQ_EINVAL);
    lora(IMQ_EINVAL, "count", [&](Call& c) { c.l.count = bad; }, IMQ_EINVAL);
    lora(IMQ_EINVAL, "max_rank", [&](Call& c) { c.l.max_rank = bad; }, IMQ_EINVAL);
  }
  lora(IMQ_EHIP, "k 2^25", [](Call& c) { c.k = 1 << 25; }, IMQ_OK);
  lora(IMQ_EUNSUPPORTED, "k past 2^25", [](Call& c) { c.k = (1 << 25) + 64; }, IMQ_EUNSUPPORTED);
  lora(IMQ_EINVAL, "k 96", [](Call& c) { c.k = 96; }, IMQ_EINVAL);
  for (int bad : {-16, 8, 63}) lora(IMQ_EINVAL, "rows", [&](Call& c) { c.l.rows = bad; }, IMQ_EINVAL);
  for (int bad : {8, 33}) lora(IMQ_EINVAL, "max_rank", [&](Call& c) { c.l.max_rank = bad; }, IMQ_EINVAL);
  lora(IMQ_EINVAL, "null a", [](Call& c) { c.l.a = nullptr; }, IMQ_EINVAL);
  lora(IMQ_EINVAL, "null b", [](Call& c) { c.l.b = nullptr; }, IMQ_EINVAL);
  lora(IMQ_EINVAL, "null first", [](Call& c) { c.l.first = nullptr; }, IMQ_EINVAL);
  lora(IMQ_EINVAL, "null scale", [](Call& c) { c.l.scale = nullptr; }, IMQ_EINVAL);
  lora(IMQ_EINVAL, "odd a", [](Call& c) { c.l.a = mem + 8; }, IMQ_EINVAL);
  lora(IMQ_EINVAL, "odd b", [](Call& c) { c.l.b = mem + 2; }, IMQ_EINVAL);
  lora(IMQ_EINVAL, "odd first", [](Call& c) { c.l.first = reinterpret_cast<int32_t*>(mem + 2); }, IMQ_EINVAL);
  lora(IMQ_EINVAL, "null which", [](Call& c) { c.which = nullptr; });
  lora(IMQ_EINVAL, "odd which", [](Call& c) { c.which = reinterpret_cast<int32_t*>(mem + 1); });
  lora(IMQ_EINVAL, "null w", [](Call& c) { c.w = nullptr; });
  lora(IMQ_EINVAL, "null x", [](Call& c) { c.x = nullptr; });
  lora(IMQ_EINVAL, "null y", [](Call& c) { c.y = nullptr; });
  lora(IMQ_EINVAL, "odd x", [](Call& c) { c.x = mem + 2; });
  lora(IMQ_EINVAL, "y is x", [](Call& c) { c.y = const_cast<void*>(c.x); });
  lora(IMQ_EINVAL, "no workspace", [](Call& c) { c.ws = nullptr; });
  lora(IMQ_EINVAL, "odd workspace", [](Call& c) { c.ws = mem + 4; });
  lora(IMQ_EINVAL, "a short workspace", [](Call& c) { c.bytes = 15; });
  Call c;
  size_t need;
  checks += 4;
  if (imq_qmm_lora_workspace(nullptr, &c.l, 64, 1, 1, IMQ_F16, &need) != IMQ_EINVAL ||
      imq_qmm_lora_workspace(&ctx, nullptr, 64, 1, 1, IMQ_F16, &need) != IMQ_EINVAL ||
      imq_qmm_lora_workspace(&ctx, &c.l, 64, 1, 1, IMQ_F16, nullptr) != IMQ_EINVAL ||
      imq_qmm_lora(nullptr, c.w, c.s, c.b, c.x, &c.l, c.which, c.y, 64, 1, 1, 64, 4, IMQ_F16, c.ws, c.bytes,
                   nullptr) != IMQ_EINVAL) {
    fprintf(stderr, "lora_refusals: null arguments\n");
    return 4;
  }
  printf("lora_refusals: %d checks\n", checks);
  return 0;
}
