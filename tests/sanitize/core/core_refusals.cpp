// core_refusals.cpp -- the argument checks of imq_core.h's entry points in a
// host-only sanitized build (TEST INFRASTRUCTURE ONLY; no GPU).
//
// Every call goes to a context of a device that does not exist: arguments that
// the checks let through fail at hipSetDevice (IMQ_EHIP), refused ones before
// that.  Prints "core_refusals: <n> checks"; any wrong status ends it.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <initializer_list>
#include <limits>
#include <random>

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
AttnPlan attention_plan(const AttnArgs&, int) { return AttnPlan{IMQ_ATTENTION_ROWS, 1, 1, 0, 0, 0}; }
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
    fprintf(stderr, "core_refusals: %s returned %d, expected %d (%s)\n", what, got, want,
            imq_last_error(&ctx));
    exit(4);
  }
}

const float kNan = std::numeric_limits<float>::quiet_NaN();
const float kInf = std::numeric_limits<float>::infinity();

imq_attention_args good() {
  imq_attention_args a{};
  a.q = a.k = a.v = mem;
  a.out = mem + 2048;
  a.q_seq = a.out_seq = 512, a.q_row = a.out_row = 128, a.q_head = a.out_head = 64;
  a.k_seq = a.v_seq = 640, a.k_row = a.v_row = 64, a.k_head = a.v_head = 64;
  a.n_seq = 2, a.heads = 2, a.kv_heads = 1, a.dim = 64, a.max_q = 4, a.max_k = 10;
  a.scale = 0.125f;
  a.dtype = IMQ_F16;
  return a;
}

template <class F>
void attention(int want, const char* what, F change) {
  imq_attention_args a = good();
  change(a);
  expect(imq_attention(&ctx, &a, nullptr), want, what);
  imq_attention_plan_info info;
  if (want != IMQ_EHIP && want != IMQ_OK)
    expect(imq_attention_plan(&ctx, &a, &info), want, what);
  else
    expect(imq_attention_plan(&ctx, &a, &info), IMQ_OK, what);
}

void attention_checks() {
  using A = imq_attention_args;
  auto* i32 = reinterpret_cast<int32_t*>(mem);
  auto* f32 = reinterpret_cast<float*>(mem);
  attention(IMQ_EHIP, "good", [](A&) {});
  attention(IMQ_EHIP, "bf16", [](A& a) { a.dtype = IMQ_BF16; });
  attention(IMQ_EHIP, "dim 1", [](A& a) { a.dim = 1; });
  attention(IMQ_EHIP, "dim 256", [](A& a) { a.dim = 256, a.out_head = 256, a.out_row = 512, a.out_seq = 2048; });
  attention(IMQ_EHIP, "keys broadcast", [](A& a) { a.k_seq = a.v_seq = a.k_row = 0; });
  attention(IMQ_EHIP, "one row at stride 0", [](A& a) { a.max_q = 1, a.out_row = 0; });
  attention(IMQ_EHIP, "slopes", [&](A& a) { a.slopes = f32; });
  attention(IMQ_EHIP, "prefix", [&](A& a) { a.causal = 1, a.prefix_lens = i32; });
  attention(IMQ_EHIP, "packed", [&](A& a) { a.q_offsets = a.k_offsets = i32, a.q_rows = 8, a.k_rows = 20, a.out_seq = 0; });
  attention(IMQ_EHIP, "no keys", [](A& a) { a.max_k = 0, a.k = a.v = nullptr; });
  attention(IMQ_OK, "no sequences", [](A& a) { a.n_seq = 0, a.q = nullptr; });
  attention(IMQ_OK, "no queries", [](A& a) { a.max_q = 0, a.out = nullptr; });
  attention(IMQ_OK, "no packed rows", [&](A& a) { a.q_offsets = i32, a.q_rows = 0; });
  attention(IMQ_EUNSUPPORTED, "f32", [](A& a) { a.dtype = IMQ_F32; });
  attention(IMQ_EUNSUPPORTED, "no dtype", [](A& a) { a.dtype = 9; });
  attention(IMQ_EUNSUPPORTED, "dim 257", [](A& a) { a.dim = 257; });
  for (int bad : {0, -1, -64}) attention(IMQ_EINVAL, "dim", [&](A& a) { a.dim = bad; });
  for (int bad : {-1, INT32_MIN}) {
    attention(IMQ_EINVAL, "n_seq", [&](A& a) { a.n_seq = bad; });
    attention(IMQ_EINVAL, "max_q", [&](A& a) { a.max_q = bad; });
    attention(IMQ_EINVAL, "max_k", [&](A& a) { a.max_k = bad; });
    attention(IMQ_EINVAL, "q_rows", [&](A& a) { a.q_rows = bad; });
    attention(IMQ_EINVAL, "k_rows", [&](A& a) { a.k_rows = bad; });
    attention(IMQ_EINVAL, "heads", [&](A& a) { a.heads = bad; });
    attention(IMQ_EINVAL, "kv_heads", [&](A& a) { a.kv_heads = bad; });
    attention(IMQ_EINVAL, "causal", [&](A& a) { a.causal = bad; });
  }
  attention(IMQ_EINVAL, "kv_heads 0", [](A& a) { a.kv_heads = 0; });
  attention(IMQ_EINVAL, "5 heads of 2", [](A& a) { a.heads = 5, a.kv_heads = 2; });
  for (float bad : {0.f, -1.f, kNan, kInf, -kInf}) attention(IMQ_EINVAL, "scale", [&](A& a) { a.scale = bad; });
  for (float bad : {-1.f, kNan, kInf}) attention(IMQ_EINVAL, "softcap", [&](A& a) { a.softcap = bad; });
  attention(IMQ_EHIP, "largest softcap", [](A& a) { a.softcap = 4096.f; });
  for (float bad : {4097.f, 3e38f}) attention(IMQ_EUNSUPPORTED, "softcap", [&](A& a) { a.softcap = bad; });
  attention(IMQ_EINVAL, "scale past fp32", [](A& a) { a.scale = 3e38f; });
  attention(IMQ_EINVAL, "scale over softcap", [](A& a) { a.scale = 1e20f, a.softcap = 1e-20f; });
  attention(IMQ_EINVAL, "out is q", [](A& a) { a.out = const_cast<void*>(a.q); });
  attention(IMQ_EINVAL, "out is v", [](A& a) { a.q = mem + 1024, a.k = mem + 512, a.out = const_cast<void*>(a.v); });
  attention(IMQ_EINVAL, "prefix without causal", [&](A& a) { a.prefix_lens = i32; });
  attention(IMQ_EINVAL, "q_offsets and q_lens", [&](A& a) { a.q_offsets = a.q_lens = i32, a.q_rows = 4; });
  attention(IMQ_EINVAL, "k_offsets and k_lens", [&](A& a) { a.k_offsets = a.k_lens = i32, a.k_rows = 4; });
  for (auto member : {&A::q_seq, &A::q_row, &A::q_head, &A::k_seq, &A::k_row, &A::k_head, &A::v_seq, &A::v_row,
                      &A::v_head, &A::out_seq, &A::out_row, &A::out_head})
    for (int64_t bad : {(int64_t)-1, INT64_MIN, INT64_MAX}) {
      attention(IMQ_EINVAL, "stride", [&](A& a) {
        a.heads = a.kv_heads = 2;
        a.out_head = 64;
        a.*member = bad;
      });
    }
  attention(IMQ_EINVAL, "outputs on each other (heads)", [](A& a) { a.out_head = 63; });
  attention(IMQ_EINVAL, "outputs on each other (rows)", [](A& a) { a.out_row = 0; });
  attention(IMQ_EINVAL, "outputs on each other (sequences)", [](A& a) { a.out_seq = 0; });
  for (auto member : {&A::q, &A::k, &A::v}) {
    attention(IMQ_EINVAL, "null", [&](A& a) { a.*member = nullptr; });
    attention(IMQ_EINVAL, "odd address", [&](A& a) { a.*member = mem + 1; });
  }
  attention(IMQ_EINVAL, "null out", [](A& a) { a.out = nullptr; });
  attention(IMQ_EINVAL, "odd out", [](A& a) { a.out = mem + 1; });
  for (auto member : {&A::q_offsets, &A::k_offsets, &A::q_lens, &A::k_lens})
    attention(IMQ_EINVAL, "misaligned lengths", [&](A& a) { a.*member = reinterpret_cast<int32_t*>(mem + 2); });
  attention(IMQ_EINVAL, "misaligned slopes", [](A& a) { a.slopes = reinterpret_cast<float*>(mem + 2); });
  expect(imq_attention(&ctx, nullptr, nullptr), IMQ_EINVAL, "null arguments");
  A a = good();
  expect(imq_attention_plan(&ctx, &a, nullptr), IMQ_EINVAL, "null plan");
}

void rope_checks() {
  const imq_rope_heads ok{mem, mem + 2048, 2, 128, 64, 128, 64, nullptr};
  auto* pos = reinterpret_cast<int32_t*>(mem);
  auto* freq = reinterpret_cast<double*>(mem);
  auto call = [&](int want, const char* what, imq_rope_heads g, int n = 1, int rows = 4, int dim = 64, int rot = 64,
                  int inter = 0, int axes = 1, const int* sec = nullptr, float amp = 1.f, float eps = 1e-6f,
                  imq_dtype t = IMQ_BF16) {
    const imq_rope_heads two[2] = {ok, g};
    expect(imq_rope(&ctx, n == 2 ? two : &g, n, rows, dim, rot, inter, pos, axes, sec, freq, amp, eps, t, nullptr),
           want, what);
  };
  auto with = [&](auto change) {
    imq_rope_heads g = ok;
    change(g);
    return g;
  };
  using G = imq_rope_heads;
  const int two_axes[2] = {20, 12}, bad_sum[2] = {20, 13}, minus[2] = {40, -8}, wide[2] = {33, -1};
  call(IMQ_EHIP, "good", ok);
  call(IMQ_EHIP, "two groups", ok, 2);
  call(IMQ_EHIP, "axes", ok, 1, 4, 64, 64, 1, 2, two_axes);
  call(IMQ_EHIP, "in place", with([](G& g) { g.y = mem; }));
  call(IMQ_EHIP, "no rows", ok, 1, 0);
  call(IMQ_EHIP, "no rotation", ok, 1, 4, 64, 0);
  call(IMQ_EINVAL, "0 groups", ok, 0);
  call(IMQ_EINVAL, "3 groups", ok, 3);
  call(IMQ_EINVAL, "rows", ok, 1, -1);
  for (int d : {0, -2, 63}) call(IMQ_EINVAL, "dim", ok, 1, 4, d, 0);
  call(IMQ_EUNSUPPORTED, "dim 1026", ok, 1, 4, 1026, 0);
  for (int r : {-2, 63, 66}) call(IMQ_EINVAL, "rot", ok, 1, 4, 64, r);
  call(IMQ_EINVAL, "interleaved", ok, 1, 4, 64, 64, 2);
  for (int x : {0, 5, 2}) call(IMQ_EINVAL, "axes", ok, 1, 4, 64, 64, 0, x);
  for (const int* s : {bad_sum, minus, wide}) call(IMQ_EINVAL, "sections", ok, 1, 4, 64, 64, 0, 2, s);
  call(IMQ_EINVAL, "amplitude", ok, 1, 4, 64, 64, 0, 1, nullptr, kNan);
  for (float e : {-1.f, kNan, kInf}) call(IMQ_EINVAL, "eps", ok, 1, 4, 64, 64, 0, 1, nullptr, 1.f, e);
  call(IMQ_EUNSUPPORTED, "dtype", ok, 1, 4, 64, 64, 0, 1, nullptr, 1.f, 0.f, (imq_dtype)3);
  for (int n : {1, 2}) {
    call(IMQ_EINVAL, "heads", with([](G& g) { g.heads = -1; }), n);
    call(IMQ_EINVAL, "null x", with([](G& g) { g.x = nullptr; }), n);
    call(IMQ_EINVAL, "null y", with([](G& g) { g.y = nullptr; }), n);
    call(IMQ_EINVAL, "odd x", with([](G& g) { g.x = mem + 1; }), n);
    call(IMQ_EINVAL, "misaligned weight", with([](G& g) { g.weight = reinterpret_cast<float*>(mem + 2); }), n);
    call(IMQ_EINVAL, "y heads on each other", with([](G& g) { g.y_head = 63; }), n);
    call(IMQ_EINVAL, "y rows on each other", with([](G& g) { g.y_row = 0; }), n);
    call(IMQ_EINVAL, "in place, other strides", with([](G& g) { g.y = mem, g.y_row = 192; }), n);
    for (auto member : {&G::x_row, &G::x_head, &G::y_row, &G::y_head})
      for (int64_t bad : {(int64_t)-1, INT64_MIN, INT64_MAX})
        call(IMQ_EINVAL, "stride", with([&](G& g) { g.*member = bad; }), n);
  }
  expect(imq_rope(&ctx, nullptr, 1, 4, 64, 64, 0, pos, 1, nullptr, freq, 1.f, 0.f, IMQ_F16, nullptr), IMQ_EINVAL,
         "null groups");
  expect(imq_rope(&ctx, &ok, 1, 4, 64, 64, 0, nullptr, 1, nullptr, freq, 1.f, 0.f, IMQ_F16, nullptr), IMQ_EINVAL,
         "null positions");
  expect(imq_rope(&ctx, &ok, 1, 4, 64, 64, 0, pos, 1, nullptr, nullptr, 1.f, 0.f, IMQ_F16, nullptr), IMQ_EINVAL,
         "null frequencies");
  expect(imq_rope(&ctx, &ok, 1, 4, 64, 64, 0, pos, 1, nullptr, reinterpret_cast<double*>(mem + 4), 1.f, 0.f, IMQ_F16,
                  nullptr), IMQ_EINVAL, "misaligned frequencies");
}

void ln_mod_checks() {
  auto* f = reinterpret_cast<float*>(mem);
  auto call = [&](int want, const char* what, const void* x = mem, imq_dtype xt = IMQ_F32, const float* sh = nullptr,
                  const int32_t* sets = nullptr, int n = 1, void* y = mem + 2048, imq_dtype yt = IMQ_F16, int rows = 2,
                  int cols = 8, float eps = 0.f, float post = 1.f) {
    expect(imq_ln_mod(&ctx, x, xt, sh, f, sets, n, y, yt, rows, cols, eps, post, nullptr), want, what);
  };
  auto* i32 = reinterpret_cast<int32_t*>(mem);
  call(IMQ_EHIP, "good", mem, IMQ_F32, f);
  call(IMQ_EHIP, "sets", mem, IMQ_F16, f, i32, 3);
  call(IMQ_EHIP, "in place", mem, IMQ_F16, f, nullptr, 1, mem);
  call(IMQ_OK, "no rows", nullptr, IMQ_F32, nullptr, nullptr, 1, nullptr, IMQ_F16, 0);
  call(IMQ_EINVAL, "null shift");
  call(IMQ_EINVAL, "null x", nullptr, IMQ_F32, f);
  call(IMQ_EINVAL, "null y", mem, IMQ_F32, f, nullptr, 1, nullptr);
  call(IMQ_EINVAL, "x off 4", mem + 2, IMQ_F32, f);
  call(IMQ_EINVAL, "y off 2", mem, IMQ_F32, f, nullptr, 1, mem + 1);
  call(IMQ_EINVAL, "in place of another type", mem, IMQ_F32, f, nullptr, 1, mem);
  call(IMQ_EINVAL, "two modulations, no sets", mem, IMQ_F32, f, nullptr, 2);
  call(IMQ_EINVAL, "no modulations", mem, IMQ_F32, f, i32, 0);
  call(IMQ_EINVAL, "rows", mem, IMQ_F32, f, nullptr, 1, mem + 64, IMQ_F16, -1);
  call(IMQ_EINVAL, "cols", mem, IMQ_F32, f, nullptr, 1, mem + 64, IMQ_F16, 1, 0);
  for (float e : {-1.f, kNan, kInf}) call(IMQ_EINVAL, "eps", mem, IMQ_F32, f, nullptr, 1, mem + 64, IMQ_F16, 1, 8, e);
  for (float p : {kNan, kInf}) call(IMQ_EINVAL, "post", mem, IMQ_F32, f, nullptr, 1, mem + 64, IMQ_F16, 1, 8, 0.f, p);
  call(IMQ_EUNSUPPORTED, "f32 out", mem, IMQ_F32, f, nullptr, 1, mem + 64, IMQ_F32);
  call(IMQ_EUNSUPPORTED, "bf16 to f16", mem, IMQ_BF16, f);
}

}  // namespace

int main() {
  ctx.device = 1 << 20;  // no such device
  ctx.cus = 256;
  attention_checks();
  rope_checks();
  ln_mod_checks();
  imq_attention_args a = good();
  imq_attention_plan_info info;
  imq_rope_heads g{};
  if (imq_attention(nullptr, &a, nullptr) != IMQ_EINVAL || imq_attention_plan(nullptr, &a, &info) != IMQ_EINVAL ||
      imq_rope(nullptr, &g, 1, 1, 2, 2, 0, nullptr, 1, nullptr, nullptr, 1.f, 0.f, IMQ_F16, nullptr) != IMQ_EINVAL ||
      imq_ln_mod(nullptr, mem, IMQ_F16, nullptr, nullptr, nullptr, 1, mem, IMQ_F16, 1, 1, 0.f, 1.f, nullptr) !=
          IMQ_EINVAL)
    return 4;
  printf("core_refusals: %d checks\n", checks);
  return 0;
}
