// attention.hip -- softmax attention (include/imq_core.h): plans and launches.
#include "attention.hpp"
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

template <int T>
hipError_t launch_t(const AttnArgs& a, hipStream_t stream) {
  const bool cap = a.softcap > 0.f, slope = a.slopes != nullptr;
  if (cap && slope) return launch_rows<T, true, true>(a, stream);
  if (cap) return launch_rows<T, true, false>(a, stream);
  if (slope) return launch_rows<T, false, true>(a, stream);
  return launch_rows<T, false, false>(a, stream);
}

}  // namespace

AttnPlan attention_plan(const AttnArgs&, int) {
  return AttnPlan{IMQ_ATTENTION_ROWS, 1, 1, 0, 0};
}

hipError_t launch_attention(const AttnArgs& a, const AttnPlan&, float*, int dtype,
                            hipStream_t stream) {
  switch (dtype) {
    case kBf16: return launch_t<kBf16>(a, stream);
    case kF16: return launch_t<kF16>(a, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace imq
