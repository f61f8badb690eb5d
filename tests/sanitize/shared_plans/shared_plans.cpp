// shared_plans.cpp -- what attention_shared_plan chooses on 256 CUs, on both sides of its rules,
// and, for sizes at random, that ranges and tiles cover every key and row once within the workspace
// (TEST INFRASTRUCTURE ONLY; no GPU).
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <random>

#include "core_kernels.hpp"
#include "imq_core.h"

namespace {

using imq::AttnArgs;
using imq::AttnShared;
using imq::SharedPlan;

int checks = 0;
const int32_t offsets[1] = {0};
alignas(16) char keys[16];

AttnArgs args(int n, int q, int k, int heads, int kv, int dim, bool packed = false) {
  AttnArgs a{};
  a.n_seq = n, a.max_q = q, a.max_k = k, a.heads = heads, a.kv_heads = kv, a.dim = dim, a.causal = 1;
  a.q_head = a.k_head = a.v_head = a.out_head = dim;
  a.q_row = a.out_row = (int64_t)heads * dim, a.k_row = a.v_row = (int64_t)kv * dim;
  if (packed) {
    a.q_offsets = a.k_offsets = offsets;
    a.q_rows = n * q, a.k_rows = n * k;
  } else {
    a.q_seq = a.out_seq = q * a.q_row, a.k_seq = a.v_seq = k * a.k_row;
    a.q_rows = q, a.k_rows = k;
  }
  a.scale = 1.f;
  return a;
}

AttnShared shared(const AttnArgs& a, int rows) {
  return AttnShared{keys, keys, (int64_t)a.kv_heads * a.dim, a.dim, (int64_t)a.kv_heads * a.dim, a.dim, rows};
}

void need(bool ok, const char* what, const AttnArgs& a, int rows, const SharedPlan& p) {
  ++checks;
  if (ok) return;
  fprintf(stderr, "shared_plans: %s: %d x %d + %d keys, %d / %d heads of %d, %d shared: kernel %d, tiles %d x %d of %d, "
          "stream %d x %d, %d of %d, %d of %d, %zu bytes\n", what, a.n_seq, a.max_q, a.max_k, a.heads, a.kv_heads, a.dim,
          rows, p.kernel, p.tiles.tile_rows, p.tiles.splits, p.tiles.chunk, p.s_tiles, p.s_rows, p.s_splits, p.s_chunk,
          p.o_splits, p.o_chunk, p.bytes);
  exit(4);
}

bool covers(int ranges, int64_t chunk, int64_t keys, int step) {
  return ranges == 0 ? keys == 0 : chunk > 0 && chunk % step == 0 && ranges * chunk >= keys && (ranges - 1) * chunk < keys;
}

SharedPlan sound(const AttnArgs& a, int rows, bool workspace) {
  const SharedPlan p = imq::attention_shared_plan(a, shared(a, rows), 256, workspace);
  const int64_t group = a.heads / a.kv_heads, of_seq = a.max_q * group, hs = (int64_t)a.n_seq * a.kv_heads;
  const int64_t columns = (a.dim > 64 ? 128 : 64) + 2;
  if (!workspace) need(p.bytes == 0, "bytes without a workspace", a, rows, p);
  if (p.kernel == IMQ_SHARED_STREAM) {
    need(of_seq <= 32, "rows of a sequence", a, rows, p);
    need((p.s_rows == 32 || p.s_rows == 64) && (int64_t)p.s_tiles * p.s_rows >= a.n_seq * of_seq &&
             (int64_t)(p.s_tiles - 1) * p.s_rows < a.n_seq * of_seq, "rows of the batch", a, rows, p);
    need(covers(p.s_splits, p.s_chunk, rows, 128) && covers(p.o_splits, p.o_chunk, a.max_k, 128), "ranges", a, rows, p);
    need(p.bytes == (size_t)((p.s_splits + p.o_splits) * hs * of_seq * columns * 4), "bytes", a, rows, p);
    need((a.kv_heads * (int64_t)p.s_tiles * p.s_splits + hs * p.o_splits) * 256 < (int64_t)1 << 32, "launch", a, rows, p);
  } else if (p.kernel == IMQ_SHARED_PACKED) {
    const int64_t line = a.q_offsets ? a.q_rows : (int64_t)a.n_seq * a.max_q;
    need(p.s_rows == 128 && (int64_t)p.s_tiles * 128 >= line * group && line * group < (int64_t)1 << 31, "rows", a, rows, p);
    need(covers(p.s_splits, p.s_chunk, rows, 64), "ranges", a, rows, p);
    need(p.bytes == (size_t)(p.s_splits * a.kv_heads * (int64_t)p.s_tiles * 128 * columns * 4), "bytes", a, rows, p);
  } else if (p.kernel == IMQ_SHARED_TILES) {
    const int64_t tiles = (of_seq + p.tiles.tile_rows - 1) / p.tiles.tile_rows;
    need(p.tiles.tile_rows == 64 || p.tiles.tile_rows == 128, "tile", a, rows, p);
    need(p.own0 % 128 == 0 && p.own0 >= rows && p.own0 - rows < 128, "first own key", a, rows, p);
    if (p.tiles.splits > 1) {
      need(covers(p.tiles.splits, p.tiles.chunk, p.own0 + a.max_k, 128), "ranges", a, rows, p);
      need(p.bytes == (size_t)(p.tiles.splits * hs * tiles * p.tiles.tile_rows * columns * 4), "bytes", a, rows, p);
    } else {
      need(p.tiles.first >= 0 && p.tiles.near_hs >= 1, "order", a, rows, p);
    }
    need(hs * tiles * p.tiles.splits * 256 < (int64_t)1 << 32, "launch", a, rows, p);
  }
  return p;
}

void expect(const char* what, const AttnArgs& a, int rows, int kernel, int tile_rows) {
  const SharedPlan p = sound(a, rows, true);
  const int got = kernel == IMQ_SHARED_TILES ? p.tiles.tile_rows : kernel == IMQ_SHARED_ROWS ? 0 : p.s_rows;
  need(p.kernel == kernel && got == tile_rows, what, a, rows, p);
}

}  // namespace

int main() {
  expect("32 rows of the batch", args(8, 1, 256, 32, 8, 128), 8192, IMQ_SHARED_STREAM, 32);
  expect("33, keys past the L2s", args(9, 1, 256, 32, 8, 128), 8192, IMQ_SHARED_STREAM, 64);
  expect("keys of 16 MiB", args(9, 1, 256, 32, 8, 128), 4096, IMQ_SHARED_STREAM, 32);
  expect("a key more", args(9, 1, 256, 32, 8, 128), 4097, IMQ_SHARED_STREAM, 64);
  expect("15 tiles of 64 rows", args(240, 1, 256, 32, 8, 128), 4096, IMQ_SHARED_STREAM, 32);
  expect("16", args(256, 1, 256, 32, 8, 128), 4096, IMQ_SHARED_STREAM, 64);
  expect("32 rows a sequence", args(4, 8, 64, 32, 8, 128), 1000, IMQ_SHARED_STREAM, 32);
  expect("36", args(4, 9, 64, 32, 8, 128), 1000, IMQ_SHARED_TILES, 64);
  expect("prompts", args(16, 512, 512, 32, 8, 128), 1024, IMQ_SHARED_TILES, 128);
  expect("short documents", args(61, 128, 128, 8, 2, 64, true), 3001, IMQ_SHARED_TILES, 128);
  expect("documents of few rows", args(61, 40, 40, 8, 2, 64, true), 3001, IMQ_SHARED_PACKED, 128);
  expect("behind 511 keys", args(61, 40, 40, 8, 2, 64, true), 511, IMQ_SHARED_TILES, 128);
  expect("behind 512", args(61, 40, 40, 8, 2, 64, true), 512, IMQ_SHARED_PACKED, 128);
  expect("a batch of 36 rows", args(64, 9, 200, 32, 8, 128), 8192, IMQ_SHARED_PACKED, 128);
  expect("of 80", args(64, 20, 200, 32, 8, 128), 8192, IMQ_SHARED_PACKED, 128);
  expect("of 84", args(64, 21, 200, 32, 8, 128), 8192, IMQ_SHARED_TILES, 128);
  expect("of 160", args(64, 40, 200, 32, 8, 128), 8192, IMQ_SHARED_PACKED, 128);
  expect("half as many own keys", args(64, 9, 512, 32, 8, 128), 1024, IMQ_SHARED_PACKED, 128);
  expect("one more", args(64, 9, 513, 32, 8, 128), 1024, IMQ_SHARED_TILES, 128);
  AttnArgs apart = args(64, 9, 200, 32, 8, 128);
  apart.q_seq += apart.q_row;
  expect("rows between the sequences", apart, 8192, IMQ_SHARED_TILES, 128);
  expect("heads of 136", args(4, 1, 64, 8, 2, 136), 100, IMQ_SHARED_ROWS, 0);
  expect("heads of 68", args(4, 1, 64, 8, 2, 68), 100, IMQ_SHARED_ROWS, 0);

  std::mt19937 rng(7);
  auto draw = [&](int lo, int hi) {  // evenly over powers
    return (int)(lo * std::exp2(std::uniform_real_distribution<>(0, std::log2((double)hi / lo))(rng)) + 0.5);
  };
  for (int i = 0; i < 20000; ++i) {
    const int kv = draw(1, 16), dim = 8 * draw(1, 16), q = draw(1, 1 << 13);
    const AttnArgs a = args(draw(1, 1 << 12), q, draw(1, 1 << 18) - 1, kv * draw(1, 16), kv, dim, i % 3 == 0);
    sound(a, draw(1, 1 << 22), i % 4 != 0);
  }
  printf("shared_plans: %d checks\n", checks);
  return 0;
}
