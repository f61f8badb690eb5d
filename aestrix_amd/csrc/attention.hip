// attention.hip -- softmax attention (include/imq_core.h): plans and launches.
#include "attention.hpp"
#include "attention_few.hpp"
#include "attention_tiles.hpp"
#include "imq_core.h"

#include <algorithm>

namespace imq {
namespace {

constexpr int kThreads = 256;

template <int T, bool kCap, bool kSlope>
__global__ __launch_bounds__(kThreads) void attn_rows_kernel(AttnArgs a) {
  __shared__ float qs[kThreads / 64][256];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t items = (int64_t)a.n_seq * a.max_q * a.heads;
  for (int64_t item = (int64_t)blockIdx.x * (kThreads / 64) + wave; item < items;
       item += (int64_t)gridDim.x * (kThreads / 64)) {
    const int head = (int)(item % a.heads);
    const int64_t row = item / a.heads;
    const int t = (int)(row % a.max_q);
    const AttnSeq s = attn_seq(a, (int)(row / a.max_q));
    if (t >= s.nq) continue;
    attn_row<T, kCap, kSlope>(a, s, head, t, attn_seen(a, s, t), qs[wave]);
  }
}

template <int T, bool kCap, bool kSlope>
hipError_t launch_rows(const AttnArgs& a, hipStream_t stream) {
  const int64_t items = (int64_t)a.n_seq * a.max_q * a.heads;
  const int64_t blocks = (items + kThreads / 64 - 1) / (kThreads / 64);
  const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)));
  hipLaunchKernelGGL((attn_rows_kernel<T, kCap, kSlope>), grid, dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

// all: rows of all tiles.
template <int T, int D, bool kCap, bool kSlope>
void launch_join(const AttnArgs& a, const AttnPlan& plan, int tile_rows, int tiles, int64_t all,
                 const float* ws, hipStream_t stream) {
  if (plan.splits > 4)
    hipLaunchKernelGGL((attn_join_kernel<T, D, 16, kCap, kSlope>), dim3((unsigned)all), dim3(256), 0,
                       stream, a, tile_rows, tiles, plan.splits, plan.chunk, ws);
  else
    hipLaunchKernelGGL((attn_join_kernel<T, D, 1, kCap, kSlope>), dim3((unsigned)((all + 15) / 16)),
                       dim3(256), 0, stream, a, tile_rows, tiles, plan.splits, plan.chunk, ws);
}

template <int T, int D, int WM, bool kCap, bool kSlope>
hipError_t launch_tiles(const AttnArgs& a, const AttnPlan& plan, float* ws, hipStream_t stream) {
  constexpr int kRows = WM * 32;
  const int64_t rows = (int64_t)a.max_q * (a.heads / a.kv_heads);
  const int tiles = (int)((rows + kRows - 1) / kRows);
  const int64_t blocks = (int64_t)a.n_seq * a.kv_heads * tiles;
  const dim3 block(attn_waves(WM) * 64);
  if constexpr (WM < 8) {  // the plan splits no keys of 256 rows
    if (plan.splits > 1) {
      hipLaunchKernelGGL((attn_tiles_kernel<T, D, WM, kCap, kSlope, true>),
                         dim3((unsigned)(blocks * plan.splits)), block, 0, stream, a, tiles,
                         plan.first, 1, plan.splits, plan.chunk, ws);
      launch_join<T, D, kCap, kSlope>(a, plan, kRows, tiles, blocks * kRows, ws, stream);
      return hipGetLastError();
    }
  }
  hipLaunchKernelGGL((attn_tiles_kernel<T, D, WM, kCap, kSlope, false>), dim3((unsigned)blocks),
                     block, 0, stream, a, tiles, plan.first, plan.near_hs, 1, 0, nullptr);
  return hipGetLastError();
}

template <int T, int D, bool kCap, bool kSlope>
hipError_t launch_few(const AttnArgs& a, const AttnPlan& plan, float* ws, hipStream_t stream) {
  const int rows = a.max_q * (a.heads / a.kv_heads);
  const unsigned hs = (unsigned)(a.n_seq * a.kv_heads);
  const dim3 block(kFewWaves * 64);
  if (plan.splits > 1) {
    hipLaunchKernelGGL((attn_few_kernel<T, D, kCap, kSlope, true>), dim3(hs * plan.splits), block, 0,
                       stream, a, rows, plan.splits, plan.chunk, ws);
    launch_join<T, D, kCap, kSlope>(a, plan, rows, 1, (int64_t)hs * rows, ws, stream);
  } else {
    hipLaunchKernelGGL((attn_few_kernel<T, D, kCap, kSlope, false>), dim3(hs), block, 0, stream, a,
                       rows, 1, 0, nullptr);
  }
  return hipGetLastError();
}

template <int T, bool kCap, bool kSlope>
hipError_t launch_scored(const AttnArgs& a, const AttnPlan& plan, float* ws, hipStream_t stream) {
  if (plan.kernel == IMQ_ATTENTION_ROWS) return launch_rows<T, kCap, kSlope>(a, stream);
  if (plan.kernel == IMQ_ATTENTION_FEW)
    return a.dim > 64 ? launch_few<T, 128, kCap, kSlope>(a, plan, ws, stream)
                      : launch_few<T, 64, kCap, kSlope>(a, plan, ws, stream);
  switch (a.dim > 64 ? plan.tile_rows : -plan.tile_rows) {
    case 256: return launch_tiles<T, 128, 8, kCap, kSlope>(a, plan, ws, stream);
    case 128: return launch_tiles<T, 128, 4, kCap, kSlope>(a, plan, ws, stream);
    case 64: return launch_tiles<T, 128, 2, kCap, kSlope>(a, plan, ws, stream);
    case -256: return launch_tiles<T, 64, 8, kCap, kSlope>(a, plan, ws, stream);
    case -128: return launch_tiles<T, 64, 4, kCap, kSlope>(a, plan, ws, stream);
    case -64: return launch_tiles<T, 64, 2, kCap, kSlope>(a, plan, ws, stream);
    default: return hipErrorInvalidValue;
  }
}

template <int T>
hipError_t launch_t(const AttnArgs& a, const AttnPlan& plan, float* ws, hipStream_t stream) {
  const bool cap = a.softcap > 0.f, slope = a.slopes != nullptr;
  if (cap && slope) return launch_scored<T, true, true>(a, plan, ws, stream);
  if (cap) return launch_scored<T, true, false>(a, plan, ws, stream);
  if (slope) return launch_scored<T, false, true>(a, plan, ws, stream);
  return launch_scored<T, false, false>(a, plan, ws, stream);
}

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
    // Two a CU from 4096 keys a range: 65 rows on 100000 keys 222 us against
    // 288, 512 on 8192 98 against 105; but 256 on 2048 36 against 21.
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

hipError_t launch_attention(const AttnArgs& a, const AttnPlan& plan, float* ws, int dtype,
                            hipStream_t stream) {
  switch (dtype) {
    case kBf16: return launch_t<kBf16>(a, plan, ws, stream);
    case kF16: return launch_t<kF16>(a, plan, ws, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace imq
