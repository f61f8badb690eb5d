// attention_plan.cpp -- which kernel an attention call takes, how many rows a
// workgroup has, and how the keys are split (host code alone).
#include <algorithm>

#include "core_kernels.hpp"
#include "imq_core.h"

namespace imq {
namespace {

// Whole 16-byte pieces everywhere, and a 64-row tile within 31-bit offsets.
bool tiles_fit(const AttnArgs& a) {
  const int64_t strides = a.q_seq | a.q_row | a.q_head | a.k_seq | a.k_row | a.k_head | a.v_seq |
                          a.v_row | a.v_head | a.out_seq | a.out_row | a.out_head;
  const uintptr_t ptrs = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.out;
  const int64_t far = (int64_t)1 << 24;  // elements of a row: 64 rows stay under 2^31 bytes
  return a.dim % 8 == 0 && a.dim <= 128 && strides % 8 == 0 && ptrs % 16 == 0 && a.k_row <= far - 128 &&
         a.v_row <= far - 128;
}

}  // namespace

AttnPlan attention_plan(const AttnArgs& a, int cus) {
  const AttnPlan by_rows{IMQ_ATTENTION_ROWS, 1, 1, 0, 0, 0, 0};
  const int64_t rows = (int64_t)a.max_q * (a.heads / a.kv_heads);
  const int64_t hs = (int64_t)a.n_seq * a.kv_heads;
  if (!tiles_fit(a) || rows > (1 << 30) || a.max_k > (1 << 30) || hs > (1 << 20) ||
      rows * hs == 0)
    return by_rows;
  const int d = a.dim > 64 ? 128 : 64;
  AttnPlan p{};
  int64_t blocks, ranges, unit;  // workgroups unsplit, ranges of keys wanted, keys of the least range
  if (rows <= 32) {
    p.kernel = IMQ_ATTENTION_FEW;
    p.tile_rows = (int)rows;
    blocks = hs;
    unit = kFewWaves * kFewKeys;  // a tile for each wave
    // One workgroup a CU: 131072 keys of 8 key heads 92.8 us (5.8 TB/s), two a
    // CU 100.1, four 95.3; 8 x up to 2048 keys 9.1 / 10.0 / 11.8 (with the
    // join's 5.2 / 5.7 / 7.7 and 4.0 / 4.3 / 4.0).
    ranges = cus / blocks;
  } else {
    p.kernel = IMQ_ATTENTION_TILES;
    // 64 rows where that gives no CU a second workgroup: the waves share the
    // keys then, and a tile of 64 keys takes 0.71 us against 0.92 (512 causal
    // rows of 32 / 8 heads 11.8 us against 13.7).  More workgroups than that
    // only load K and V more often (2048 rows of 64 heads on 1024 keys 102 us
    // against 90, 1024 image rows of 24 heads 28 against 25).
    p.tile_rows = hs * ((rows + 63) / 64) > cus ? 128 : 64;
    // 256 rows where they fill the card: a workgroup of eight waves on one stage
    // of keys then writes LDS half as often as two of four.  4608 rows of 24
    // heads 279 us against 294 (64 elements 155 / 169), 1536 53 / 55, 8192 causal
    // rows of 32 / 8 heads 532 / 543, 32768 8.03 ms / 8.24.  Not where half of the
    // CUs would have none in the last round: two small ones share a CU, one alone
    // is quicker (9216 rows 1056 us against 1014); nor short causal rows, whose
    // tiles differ most (2048 62 us against 48, 4 x 2048 155 / 152).
    const int64_t wide = hs * ((rows + 255) / 256), last = wide % cus;
    if ((last == 0 || last > cus / 2) &&
        (a.causal ? rows >= 4096 && wide >= 2 * cus : rows >= 1024))
      p.tile_rows = 256;
    const int64_t tiles = (rows + p.tile_rows - 1) / p.tile_rows;
    blocks = hs * tiles;
    // (attn_tiles_kernel; four prompts of 512, 316, 121 and 437 rows, 32 / 8 heads:
    // 18.0 us against 19.4.)
    p.first = (int)(p.tile_rows < 256 && blocks <= 2 * cus && blocks > cus ? cus / hs : tiles);
    // 32 sequences and key heads at a time, so that the L2s hold what is being read
    // of K and V, where that gives 16 rounds of workgroups of one size: 128 prompts of 512
    // rows, 32 / 8 heads, 530 us against 623, 64 x 1024 of 16 655 / 762, 32 x 1024 of 32 / 8
    // 406 / 420, 256 x 512 of 12 of 64 305 / 430.  Otherwise all, tile by tile, so that the longest start first: 61 documents of
    // up to 777 rows 82 us against 102, 16 x 4096 of 8 heads of 64 306 / 326.
    const int64_t places = p.tile_rows == 256 ? cus : 2 * cus;
    const bool even = !a.q_offsets && !a.q_lens && !a.k_offsets && !a.k_lens;
    p.near_hs = (int)(even && blocks >= 16 * places ? std::min<int64_t>(hs, 32) : hs);
    unit = 4 * kAttnKeys;
    ranges = cus / blocks;
    // Two a CU from 4096 keys a range: 65 queries of 32 / 8 heads on 100000 keys 196 us
    // against 280, 512 on 8192 90 / 94; but 256 on 2048 27 / 24, and 65 of 8 / 2
    // heads on 100000, with 51 ranges for 25, 76 / 67.
    const int64_t two = 2 * cus / blocks;
    if (p.tile_rows == 256)
      ranges = 1;  // more than cus / 2 workgroups already, and one a CU
    else if (two > 1 && a.max_k / two >= 4096) ranges = two;
  }
  if (blocks * 512 >= ((int64_t)1 << 32)) return by_rows;
  ranges = std::min<int64_t>(ranges, (a.max_k + unit - 1) / unit);
  p.splits = 1;
  if (ranges > 1) {
    const int64_t step = p.kernel == IMQ_ATTENTION_FEW ? unit : kAttnKeys;
    const int64_t steps = (a.max_k + step - 1) / step, per = (steps + ranges - 1) / ranges;
    if (per < steps) {
      p.chunk = (int)(per * step);
      p.splits = (int)((steps + per - 1) / per);
      p.bytes = (size_t)p.splits * blocks * p.tile_rows * (d + 2) * 4;
    }
  }
  return p;
}

}  // namespace imq
