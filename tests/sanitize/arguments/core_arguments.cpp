// core_arguments.cpp -- combinations of arguments of imq_core.h's entry points on
// a host-only sanitized build (TEST INFRASTRUCTURE ONLY; no GPU).
//
// Every call goes to a context of a device that does not exist: arguments that
// the checks let through fail at hipSetDevice (IMQ_EHIP), refused ones before
// that.  Prints "core_arguments: <n> checks"; any wrong status ends it.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <random>
#include <vector>

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

template <class F>
void rope(int want, const char* what, int rows, F change) {
  static const double freq[32] = {};
  static const int32_t pos[64] = {};
  imq_rope_heads g{mem, mem + 2048, 2, 128, 64, 128, 64, nullptr};
  change(g);
  expect(imq_rope(&ctx, &g, 1, rows, 64, 64, 0, pos, 1, nullptr, freq, 1.f, 0.f, IMQ_BF16, nullptr), want, what);
}

// Outputs of different rows, heads and sequences at one place.
void outputs_on_each_other() {
  auto* lens = reinterpret_cast<int32_t*>(mem);
  struct Case {
    int n, rows, heads;
    int64_t seq, row, head;
    bool apart;
  };
  std::vector<Case> cases = {
      {2, 4, 2, 512, 128, 64, true},    {2, 4, 2, 256, 64, 1024, true},  // heads outermost
      {2, 4, 2, 64, 256, 128, true},    // sequences innermost
      {1, 4, 2, 0, 64, 64, false},      // the second head of a row is the next row
      {1, 4, 2, 0, 100, 64, false},     // half of it
      {1, 2, 2, 0, 128, 192, true},     // neither inside the other, and yet apart
      {1, 4, 2, 0, 128, 192, true},     {1, 4, 2, 0, 128, 256, false},  {1, 4, 2, 0, 128, 290, false},
      {1, 4, 4, 0, 128, 64, false},     {2, 4, 2, 500, 128, 64, false}, {2, 4, 2, 128, 128, 64, false},
      {3, 2, 2, 192, 576, 128, true},   {3, 2, 2, 192, 320, 128, false},
        {3, 2, 2, 128, 1000, 448, true}, {2, 1, 1, 64, 0, 0, true},
      {1, 1, 2, 0, 0, 64, true},        {1, 65000, 70, 0, 70 * 64, 64, true}, {1, 65000, 70, 0, 69 * 64, 64, false}};
  const size_t told = cases.size();
  std::mt19937 rng(5);
  for (int i = 0; i < 2000; ++i) {
    auto below = [&](int n) { return (int)(rng() % n); };
    auto stride = [&] { return below(2) ? 32 * below(40) : 64 + below(700); };
    cases.push_back({1 + below(3), 1 + below(5), 1 + below(5), stride(), stride(), stride(), true});
  }
  for (Case& c : cases) {
    // As a list of places, where there are few.
    if (c.n * c.rows * c.heads < 1000) {
      bool apart = true;
      std::vector<int64_t> at;
      for (int s = 0; s < c.n; ++s)
        for (int r = 0; r < c.rows; ++r)
          for (int h = 0; h < c.heads; ++h) at.push_back(s * c.seq + r * c.row + h * c.head);
      std::sort(at.begin(), at.end());
      for (size_t i = 1; i < at.size(); ++i) apart = apart && at[i] - at[i - 1] >= 64;
      if ((size_t)(&c - cases.data()) >= told) {
        c.apart = apart;
      } else if (apart != c.apart) {
        fprintf(stderr, "core_arguments: case %d is told wrong\n", (int)(&c - cases.data()));
        exit(4);
      }
    }
    auto strides = [&](A& a) {
      a.n_seq = c.n, a.max_q = c.rows, a.heads = c.heads;
      a.out_seq = c.seq, a.out_row = c.row, a.out_head = c.head;
    };
    attention(c.apart ? IMQ_EHIP : IMQ_EINVAL, "outputs on each other", strides);
    if (c.n == 1) {
      attention(c.apart ? IMQ_EHIP : IMQ_EINVAL, "packed outputs on each other", [&](A& a) {
        strides(a);
        a.q_offsets = a.k_offsets = lens, a.q_rows = c.rows, a.k_rows = 10, a.n_seq = 3, a.out_seq = 0;
      });
      rope(c.apart ? IMQ_EHIP : IMQ_EINVAL, "rope's outputs on each other", c.rows,
           [&](imq_rope_heads& g) { g.heads = c.heads, g.y_row = c.row, g.y_head = c.head; });
    }
  }
  // Lengths keep windows apart that would reach into each other.
  attention(IMQ_EHIP, "windows and lengths", [&](A& a) { a.out_seq = 128, a.q_lens = lens; });
  attention(IMQ_EINVAL, "rows, and lengths", [&](A& a) { a.out_row = 64, a.q_lens = lens; });
  // As many of neither kind as nothing could go through.
  attention(IMQ_EINVAL, "large strides on each other", [&](A& a) {
    a.max_q = 1 << 30, a.heads = a.kv_heads = 1 << 30, a.n_seq = 1, a.out_row = 100, a.out_head = 99;
  });
}

// A thread of 256 adds up a 256th of a row, one after another.
void long_rows() {
  auto* f = reinterpret_cast<float*>(mem);
  auto call = [&](int want, int cols, int rows) {
    expect(imq_ln_mod(&ctx, mem, IMQ_F32, f, f, nullptr, 1, mem + 2048, IMQ_F16, rows, cols, 0.f, 1.f, nullptr), want,
           "a long row");
  };
  for (int rows : {1, 3}) {
    call(IMQ_EHIP, 1 << 20, rows);
    for (int cols : {(1 << 20) + 1, 1 << 24, INT32_MAX - 255, INT32_MAX}) call(IMQ_EUNSUPPORTED, cols, rows);
  }
}

}  // namespace

int main() {
  ctx.device = 1 << 20;  // no such device
  ctx.cus = 256;
  scales_with_slopes();
  outputs_on_each_other();
  long_rows();
  printf("core_arguments: %d checks\n", checks);
  return 0;
}
