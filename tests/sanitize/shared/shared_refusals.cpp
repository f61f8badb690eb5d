// shared_refusals.cpp -- the argument checks of imq_attention_shared in a
// host-only sanitized build (TEST INFRASTRUCTURE ONLY; no GPU).
//
// Every call goes to a context of a device that does not exist: arguments that
// the checks let through fail at hipSetDevice (IMQ_EHIP), refused ones before
// that.  Prints "shared_refusals: <n> checks"; any wrong status ends it.
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
hipError_t launch_attention(const AttnArgs&, const AttnPlan&, float*, int, hipStream_t) {
  return hipErrorNoDevice;
}
hipError_t launch_attention_shared_bf16(const AttnArgs&, const AttnShared&, const SharedPlan&, float*,
                                        hipStream_t) {
  return hipErrorNoDevice;
}
hipError_t launch_attention_shared_f16(const AttnArgs&, const AttnShared&, const SharedPlan&, float*,
                                       hipStream_t) {
  return hipErrorNoDevice;
}
}  // namespace imq

namespace {

int checks = 0;
imq_ctx ctx;
alignas(16) char mem[4096];

template <class F>
void shared(int want, const char* what, F change) {
  imq_attention_args a{};
  a.q = a.k = a.v = mem;
  a.out = mem + 2048;
  a.q_seq = a.out_seq = 512, a.q_row = a.out_row = 128, a.q_head = a.out_head = 64;
  a.k_seq = a.v_seq = 640, a.k_row = a.v_row = 64, a.k_head = a.v_head = 64;
  a.n_seq = 2, a.heads = 2, a.kv_heads = 1, a.dim = 64, a.max_q = 4, a.max_k = 10;
  a.scale = 0.125f;
  a.dtype = IMQ_F16;
  imq_shared_keys s{mem, mem + 1024, 64, 64, 64, 64, 7};
  change(a, s);
  ++checks;
  const int got = imq_attention_shared(&ctx, &a, &s, nullptr);
  if (got != want || (want != IMQ_OK && strlen(imq_last_error(&ctx)) == 0)) {
    fprintf(stderr, "shared_refusals: %s returned %d, expected %d (%s)\n", what, got, want,
            imq_last_error(&ctx));
    exit(4);
  }
}

}  // namespace

int main() {
  using A = imq_attention_args;
  using S = imq_shared_keys;
  ctx.device = 1 << 20;
  shared(IMQ_EHIP, "good", [](A&, S&) {});
  shared(IMQ_EHIP, "no shared keys", [](A&, S& s) { s = S{}; });
  shared(IMQ_EHIP, "no own keys", [](A& a, S&) { a.max_k = 0, a.k = a.v = nullptr; });
  shared(IMQ_EHIP, "one row for all", [](A&, S& s) { s.k_row = s.v_row = 0; });
  shared(IMQ_EHIP, "as many keys as there may be", [](A&, S& s) { s.rows = INT32_MAX - 10; });
  shared(IMQ_OK, "no sequences", [](A& a, S& s) { a.n_seq = 0, s.k = nullptr; });
  shared(IMQ_OK, "no queries", [](A& a, S& s) { a.max_q = 0, s.v = nullptr; });
  shared(IMQ_EINVAL, "a key too many", [](A&, S& s) { s.rows = INT32_MAX - 9; });
  for (int bad : {-1, INT32_MIN}) shared(IMQ_EINVAL, "rows", [&](A&, S& s) { s.rows = bad; });
  for (auto member : {&S::k_row, &S::k_head, &S::v_row, &S::v_head})
    for (int64_t bad : {(int64_t)-1, INT64_MIN, INT64_MAX})
      shared(IMQ_EINVAL, "a stride", [&](A& a, S& s) { a.heads = a.kv_heads = 2, s.*member = bad; });
  shared(IMQ_EINVAL, "null k", [](A&, S& s) { s.k = nullptr; });
  shared(IMQ_EINVAL, "null v", [](A&, S& s) { s.v = nullptr; });
  shared(IMQ_EINVAL, "odd k", [](A&, S& s) { s.k = mem + 1; });
  shared(IMQ_EINVAL, "odd v", [](A&, S& s) { s.v = mem + 3; });
  shared(IMQ_EINVAL, "out is the shared k", [](A& a, S& s) { s.k = a.out; });
  shared(IMQ_EINVAL, "out is the shared v", [](A& a, S& s) { s.v = a.out; });
  // The other arguments' checks are imq_attention's.
  shared(IMQ_EUNSUPPORTED, "f32", [](A& a, S&) { a.dtype = IMQ_F32; });
  shared(IMQ_EINVAL, "kv_heads 0", [](A& a, S&) { a.kv_heads = 0; });
  shared(IMQ_EINVAL, "out is q", [](A& a, S&) { a.out = const_cast<void*>(a.q); });
  const imq_attention_args none{};
  checks += 3;
  if (imq_attention_shared(nullptr, &none, nullptr, nullptr) != IMQ_EINVAL ||
      imq_attention_shared(&ctx, nullptr, nullptr, nullptr) != IMQ_EINVAL ||
      imq_attention_shared(&ctx, &none, nullptr, nullptr) == IMQ_OK) {
    fprintf(stderr, "shared_refusals: null arguments\n");
    return 4;
  }
  printf("shared_refusals: %d checks\n", checks);
  return 0;
}
