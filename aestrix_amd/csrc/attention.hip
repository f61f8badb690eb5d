// attention.hip -- softmax attention (include/imq_core.h): the launches of a plan.
#include "attention.hpp"
#include "attention_few.hpp"
#include "attention_tiles.hpp"
#include "imq_core.h"

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

}  // namespace

hipError_t launch_attention(const AttnArgs& a, const AttnPlan& plan, float* ws, int dtype,
                            hipStream_t stream) {
  switch (dtype) {
    case kBf16: return launch_t<kBf16>(a, plan, ws, stream);
    case kF16: return launch_t<kF16>(a, plan, ws, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace imq
