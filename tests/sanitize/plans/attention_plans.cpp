// attention_plans.cpp -- what attention_plan chooses on 256 CUs, on both sides of
// every rule (TEST INFRASTRUCTURE ONLY; no GPU).
#include <cstdio>
#include <cstdlib>
#include <set>
#include <tuple>

#include "core_kernels.hpp"
#include "imq_core.h"

namespace {

using imq::AttnArgs;
using imq::AttnPlan;

int checks = 0;

AttnArgs args(int n, int q, int k, int heads, int kv, int dim, bool causal) {
  AttnArgs a{};
  a.n_seq = n, a.max_q = q, a.max_k = k, a.heads = heads, a.kv_heads = kv, a.dim = dim, a.causal = causal;
  a.q_head = a.k_head = a.v_head = a.out_head = dim;
  a.q_row = a.out_row = (int64_t)heads * dim, a.k_row = a.v_row = (int64_t)kv * dim;
  a.q_seq = a.out_seq = q * a.q_row, a.k_seq = a.v_seq = k * a.k_row;
  a.scale = 1.f;
  return a;
}

void expect(const char* what, const AttnArgs& a, int kernel, int tile_rows, int splits, int chunk, int first, int near_hs) {
  ++checks;
  const AttnPlan p = imq::attention_plan(a, 256);
  const int64_t rows = (int64_t)a.max_q * (a.heads / a.kv_heads), hs = (int64_t)a.n_seq * a.kv_heads;
  const int64_t tiles = kernel == IMQ_ATTENTION_TILES ? (rows + tile_rows - 1) / tile_rows : 1;
  const size_t bytes = splits > 1 ? (size_t)splits * hs * tiles * tile_rows * ((a.dim > 64 ? 128 : 64) + 2) * 4 : 0;
  if (p.kernel != kernel || p.tile_rows != tile_rows || p.splits != splits || p.chunk != chunk || p.first != first ||
      p.near_hs != near_hs || p.bytes != bytes) {
    fprintf(stderr, "attention_plans: %s: kernel %d, %d rows, %d splits of %d, first %d, near %d, %zu bytes; expected %d, "
            "%d, %d of %d, %d, %d, %zu\n", what, p.kernel, p.tile_rows, p.splits, p.chunk, p.first, p.near_hs, p.bytes,
            kernel, tile_rows, splits, chunk, first, near_hs, bytes);
    exit(4);
  }
}

void few(const char* what, const AttnArgs& a, int rows, int splits, int chunk) {
  expect(what, a, IMQ_ATTENTION_FEW, rows, splits, chunk, 0, 0);
}
void tiles(const char* what, const AttnArgs& a, int rows, int first, int near_hs, int splits = 1, int chunk = 0) {
  expect(what, a, IMQ_ATTENTION_TILES, rows, splits, chunk, first, near_hs);
}
void by_rows(const char* what, const AttnArgs& a) { expect(what, a, IMQ_ATTENTION_ROWS, 1, 1, 0, 0, 0); }

template <class F>
AttnArgs with(AttnArgs a, F change) {
  change(a);
  return a;
}

void few_rows() {
  few("one token over a long cache", args(1, 1, 131072, 32, 8, 128, true), 4, 32, 4096);
  few("eight tokens", args(8, 1, 2048, 32, 8, 128, true), 4, 4, 512);
  few("a range's keys", args(1, 1, 128, 32, 8, 128, true), 4, 1, 0);
  few("a key more", args(1, 1, 129, 32, 8, 128, true), 4, 2, 128);
  few("no keys", args(1, 1, 0, 32, 8, 128, true), 4, 1, 0);
  few("32 rows", args(1, 8, 385, 4, 1, 64, false), 32, 4, 128);
  few("ranges that do not come out even", args(100, 1, 640, 1, 1, 64, false), 1, 2, 384);
  few("fewer ranges than there could be", args(60, 1, 640, 1, 1, 64, false), 1, 3, 256);
  few("more key heads than half the CUs", args(129, 1, 9999, 1, 1, 64, false), 1, 1, 0);
  tiles("33 rows", args(1, 33, 1000, 1, 1, 128, false), 64, 1, 1, 4, 256);
  tiles("33 rows of three heads", args(1, 11, 1000, 3, 1, 72, false), 64, 1, 1, 4, 256);
}

void heights() {
  tiles("a workgroup of 64 rows a CU", args(1, 512, 512, 32, 8, 128, true), 64, 32, 8);
  tiles("one tile more", args(1, 513, 513, 32, 8, 128, true), 128, 17, 8);
  tiles("two workgroups a CU", args(4, 512, 512, 32, 8, 128, true), 128, 8, 32);
  tiles("the same, dense", args(4, 512, 512, 32, 8, 128, false), 256, 8, 32);
  tiles("1023 dense rows", args(1, 1023, 1023, 36, 36, 128, false), 128, 7, 36);
  tiles("1024 dense rows", args(1, 1024, 1024, 36, 36, 128, false), 256, 4, 36);
  tiles("half of the CUs in the last round", args(1, 1024, 1024, 32, 32, 128, false), 128, 8, 32);
  tiles("1536 rows of 24 heads", args(1, 1536, 1536, 24, 24, 128, false), 256, 6, 24);
  tiles("4608 rows of 24 heads", args(1, 4608, 4608, 24, 24, 128, false), 256, 18, 24);
  tiles("9216 rows of 24 heads", args(1, 9216, 9216, 24, 24, 128, false), 128, 72, 24);
  tiles("4095 causal rows", args(1, 4095, 4095, 32, 32, 128, true), 128, 32, 32);
  tiles("4096 causal rows", args(1, 4096, 4096, 32, 32, 128, true), 256, 16, 32);
  tiles("one round of causal rows", args(1, 8192, 8192, 8, 1, 128, true), 128, 256, 1);
  tiles("16384 causal rows", args(1, 16384, 16384, 32, 8, 128, true), 256, 256, 8);
}

void orders_and_ranges() {
  tiles("many prompts", args(128, 512, 512, 32, 8, 128, true), 128, 16, 32);
  int32_t lens = 0;
  tiles("many prompts of all lengths", with(args(128, 512, 512, 32, 8, 128, true), [&](AttnArgs& a) { a.q_lens = &lens; }), 128, 16, 1024);
  tiles("not quite as many", args(63, 512, 512, 32, 8, 128, true), 128, 16, 504);
  tiles("65 queries over a long cache", args(1, 65, 100000, 32, 8, 128, true), 64, 5, 8, 12, 8384);
  tiles("512 queries over a cache", args(1, 512, 8192, 32, 8, 128, true), 64, 32, 8, 2, 4096);
  tiles("a key less, and a range of 4095", args(1, 512, 8191, 32, 8, 128, true), 64, 32, 8);
  tiles("256 queries over a short one", args(1, 256, 2048, 32, 8, 128, true), 64, 16, 8, 2, 1024);
  tiles("a split of 128 rows", args(1, 1100, 12400, 16, 16, 128, false), 128, 9, 16, 3, 4160);
}

void unfit() {
  const AttnArgs ok = args(2, 100, 100, 4, 2, 128, true);
  tiles("fit", ok, 64, 4, 4);
  by_rows("136 elements", args(2, 100, 100, 4, 2, 136, true));
  by_rows("256 elements", args(2, 1, 100, 4, 2, 256, true));
  by_rows("100 elements", args(2, 100, 100, 4, 2, 100, true));
  by_rows("one element", args(2, 100, 100, 4, 2, 1, true));
  for (auto m : {&AttnArgs::q_seq, &AttnArgs::q_row, &AttnArgs::q_head, &AttnArgs::k_seq, &AttnArgs::k_row, &AttnArgs::k_head,
                 &AttnArgs::v_seq, &AttnArgs::v_row, &AttnArgs::v_head, &AttnArgs::out_seq, &AttnArgs::out_row,
                 &AttnArgs::out_head}) {
    by_rows("a stride off 16 bytes", with(ok, [&](AttnArgs& a) { a.*m += 4; }));
    tiles("a stride of 16 bytes more", with(ok, [&](AttnArgs& a) { a.*m += 8; }), 64, 4, 4);
  }
  for (auto m : {&AttnArgs::q, &AttnArgs::k, &AttnArgs::v})
    by_rows("an address off 16 bytes", with(ok, [&](AttnArgs& a) { a.*m = (void*)(uintptr_t)8; }));
  by_rows("an output off 16 bytes", with(ok, [&](AttnArgs& a) { a.out = (void*)(uintptr_t)8; }));
  for (auto m : {&AttnArgs::k_row, &AttnArgs::v_row}) {
    tiles("rows as far apart as 31 bits take", with(ok, [&](AttnArgs& a) { a.*m = (1 << 24) - 128; }), 64, 4, 4);
    by_rows("rows farther apart", with(ok, [&](AttnArgs& a) { a.*m = (1 << 24) - 120; }));
  }
  by_rows("no rows", args(2, 0, 100, 4, 2, 128, true));
  by_rows("no sequences", args(0, 100, 100, 4, 2, 128, true));
  few("2^20 key heads", args(1 << 20, 1, 9, 1, 1, 64, true), 1, 1, 0);
  by_rows("more than 2^20 key heads", args((1 << 20) + 1, 1, 9, 1, 1, 64, true));
  tiles("just under 2^32 threads", args(1 << 20, 1792, 64, 1, 1, 64, false), 256, 7, 32);
  by_rows("2^32 threads", args(1 << 20, 2048, 64, 1, 1, 64, false));
}

// The kernel's place of every workgroup: each sequence and key head, tile and range once.
void places() {
  for (int n : {1, 3, 40, 70, 128, 500})
    for (int q : {33, 65, 130, 512, 1000, 2100})
      for (int kv : {1, 3, 8})
        for (int keys : {q, 9000})
          for (bool causal : {false, true}) {
            const AttnArgs a = args(n, q, keys, 2 * kv, kv, 128, causal);
            const AttnPlan p = imq::attention_plan(a, 256);
            if (p.kernel != IMQ_ATTENTION_TILES) exit(4);
            const int hs_n = n * kv, tiles = (2 * q + p.tile_rows - 1) / p.tile_rows;
            const bool split = p.splits > 1;
            std::set<std::tuple<int, int, int>> seen;
            for (int b = 0; b < hs_n * tiles * p.splits; ++b) {
              const int near = split ? 1 : p.near_hs;  // as the launches pass it
              const int hs0 = split ? 0 : b / (near * tiles) * near;
              const int now = split ? hs_n : (near < hs_n - hs0 ? near : hs_n - hs0);
              const int at = b - hs0 * tiles, hs = hs0 + at % now, rest = at / now;
              const int rank = split ? rest / p.splits : rest, range = split ? rest % p.splits : 0;
              const int tile = rank < p.first ? tiles - 1 - rank : rank - p.first;
              if (hs < 0 || hs >= hs_n || tile < 0 || tile >= tiles || !seen.insert({hs, tile, range}).second) {
                fprintf(stderr, "attention_plans: workgroup %d of %d x %d rows, %d key heads: (%d, %d, %d)\n", b, n, q, kv, hs,
                        tile, range);
                exit(4);
              }
            }
            if (split && ((int64_t)p.splits * p.chunk < keys || (int64_t)(p.splits - 1) * p.chunk >= keys || p.chunk % 64)) exit(5);
            ++checks;
          }
}

}  // namespace

int main() {
  few_rows();
  heights();
  orders_and_ranges();
  unfit();
  places();
  printf("attention_plans: %d checks\n", checks);
  return 0;
}
