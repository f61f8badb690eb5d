// lora.hip -- the first product of adapters beside a projection: u = scale * A x, a row's
// adapter's (include/imq_lora.h).
#include "lora_device.hpp"

namespace imq {
namespace {

constexpr int kThreads = 256;

// A wave per row and rank.
template <int T>
__global__ __launch_bounds__(kThreads) void lora_shrink_kernel(LoraArgs l, const uint16_t* x, int k,
                                                              int m) {
  const int lane = threadIdx.x & 63;
  const int64_t items = (int64_t)m * l.max_rank, step = (int64_t)gridDim.x * (kThreads / 64);
  for (int64_t at = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6); at < items; at += step) {
    const int row = (int)(at / l.max_rank), r = (int)(at % l.max_rank);
    const int i = lora_of(l, row);
    if (i < 0) continue;
    const LoraAt to = lora_at(l, i);
    if (r >= to.rank) continue;
    const uint16_t* a = l.a + (size_t)(to.row + r) * k;
    const uint16_t* xr = x + (size_t)row * k;
    float sum = 0.f;
    for (int c = lane * 8; c < k; c += 512) {
      const uint4 av = *reinterpret_cast<const uint4*>(a + c), xv = *reinterpret_cast<const uint4*>(xr + c);
      const uint32_t aw[4] = {av.x, av.y, av.z, av.w}, xw[4] = {xv.x, xv.y, xv.z, xv.w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        sum = T == kBf16 ? dot2_bf16(aw[e], xw[e], sum) : dot2_f16(aw[e], xw[e], sum);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
    if (lane == 0) l.u[at] = sum * l.scale[i];
  }
}

}  // namespace

hipError_t launch_lora_shrink(const LoraArgs& l, const void* x, int k, int m, int dtype,
                              hipStream_t stream) {
  const int64_t blocks = ((int64_t)m * l.max_rank + kThreads / 64 - 1) / (kThreads / 64);
  const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)));
  const auto* xx = static_cast<const uint16_t*>(x);
  switch (dtype) {
    case kBf16:
      hipLaunchKernelGGL((lora_shrink_kernel<kBf16>), grid, dim3(kThreads), 0, stream, l, xx, k, m);
      break;
    case kF16:
      hipLaunchKernelGGL((lora_shrink_kernel<kF16>), grid, dim3(kThreads), 0, stream, l, xx, k, m);
      break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace imq
