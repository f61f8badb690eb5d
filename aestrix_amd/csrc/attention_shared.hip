// attention_shared.hip -- softmax attention of sequences that begin with the same keys
// (imq_attention_shared, include/imq_core.h).
#include "attention.hpp"
#include "imq_core.h"

namespace imq {
namespace {

constexpr int kThreads = 256;

template <int T, bool kCap, bool kSlope>
__global__ __launch_bounds__(kThreads) void attn_shared_rows_kernel(AttnArgs a, AttnShared sh) {
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
    attn_row<T, kCap, kSlope, true>(a, s, head, t, attn_seen(a, s, t), qs[wave], sh);
  }
}

template <int T, bool kCap, bool kSlope>
hipError_t launch_rows(const AttnArgs& a, const AttnShared& sh, hipStream_t stream) {
  const int64_t items = (int64_t)a.n_seq * a.max_q * a.heads;
  const int64_t blocks = (items + kThreads / 64 - 1) / (kThreads / 64);
  const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)));
  hipLaunchKernelGGL((attn_shared_rows_kernel<T, kCap, kSlope>), grid, dim3(kThreads), 0, stream, a,
                     sh);
  return hipGetLastError();
}

template <int T>
hipError_t launch_t(const AttnArgs& a, const AttnShared& sh, hipStream_t stream) {
  const bool cap = a.softcap > 0.f, slope = a.slopes != nullptr;
  if (cap && slope) return launch_rows<T, true, true>(a, sh, stream);
  if (cap) return launch_rows<T, true, false>(a, sh, stream);
  if (slope) return launch_rows<T, false, true>(a, sh, stream);
  return launch_rows<T, false, false>(a, sh, stream);
}

}  // namespace

hipError_t launch_attention_shared(const AttnArgs& a, const AttnShared& sh, int dtype,
                                   hipStream_t stream) {
  switch (dtype) {
    case kBf16: return launch_t<kBf16>(a, sh, stream);
    case kF16: return launch_t<kF16>(a, sh, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace imq
