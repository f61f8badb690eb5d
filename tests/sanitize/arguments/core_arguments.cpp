// core_arguments.cpp -- combinations of arguments of imq_core.h's entry points on
// a host-only sanitized build (TEST INFRASTRUCTURE ONLY; no GPU).
//
// Every call goes to a context of a device that does not exist: arguments that
// the checks let through fail at hipSetDevice (IMQ_EHIP), refused ones before
// that.  Prints "core_arguments: <n> checks"; any wrong status ends it.
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "core_kernels.hpp"
#include "ctx.hpp"
#include "imq.h"
#include "imq_core.h"

namespace imq {
hipError_t launch_ln_mod(const void*, int, const float*, const float*, const int32_t*, int, void*,
                         int, int, int, float, float, hipStream_t) {
  return hipErrorNoDevice;
}
hipError_t launch_rope(const RopeArgs&, bool, int, hipStream_t) { return hipErrorNoDevice; }
AttnPlan attention_plan(const AttnArgs&, int) { return AttnPlan{IMQ_ATTENTION_ROWS, 1, 1}; }
hipError_t launch_attention(const AttnArgs&, const AttnPlan&, float*, int, hipStream_t) {
  return hipErrorNoDevice;
}
}  // namespace imq

namespace {

int checks = 0;
imq_ctx ctx;
alignas(16) char mem[4096];

void expect(int got, int want, const char* what) {
  ++checks;
  if (got != want || (want != IMQ_OK && strlen(imq_last_error(&ctx)) == 0)) {
    fprintf(stderr, "core_arguments: %s returned %d, expected %d (%s)\n", what, got, want,
            imq_last_error(&ctx));
    exit(4);
  }
}

using A = imq_attention_args;

template <class F>
void attention(int want, const char* what, F change) {
  A a{};
  a.q = a.k = a.v = mem;
  a.out = mem + 2048;
  a.q_seq = a.out_seq = 512, a.q_row = a.out_row = 128, a.q_head = a.out_head = 64;
  a.k_seq = a.v_seq = 640, a.k_row = a.v_row = 64, a.k_head = a.v_head = 64;
  a.n_seq = 2, a.heads = 2, a.kv_heads = 1, a.dim = 64, a.max_q = 4, a.max_k = 10;
  a.scale = 0.125f;
  a.dtype = IMQ_F16;
  change(a);
  expect(imq_attention(&ctx, &a, nullptr), want, what);
}

// A slope's fall is divided by the scale within a tile.
void scales_with_slopes() {
  auto* f32 = reinterpret_cast<float*>(mem);
  for (float tiny : {1e-44f, 1e-38f, 1e-30f, 5.0e-20f}) {
    attention(IMQ_EUNSUPPORTED, "tiny scale and slopes", [&](A& a) { a.scale = tiny, a.slopes = f32; });
    attention(IMQ_EHIP, "tiny scale", [&](A& a) { a.scale = tiny; });
    attention(IMQ_EHIP, "tiny scale, capped, and slopes", [&](A& a) { a.scale = tiny, a.slopes = f32, a.softcap = 5.f; });
  }
  attention(IMQ_EHIP, "the least scale with slopes", [&](A& a) { a.scale = 0x1p-64f, a.slopes = f32; });
}

}  // namespace

int main() {
  ctx.device = 1 << 20;  // no such device
  ctx.cus = 256;
  scales_with_slopes();
  printf("core_arguments: %d checks\n", checks);
  return 0;
}
