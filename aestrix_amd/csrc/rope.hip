// rope.hip -- per-head RMSNorm and rotary positions of the query and key heads.
//
// y = turn(x * rsqrt(mean(x^2) + eps) * w) by angle_j = position * inv_freq[j]:
// the reference's dd_rmsnorm_pitched + dd_rope_interleaved
// (Sources/ImarelloDirect/DirectDiTKernels.swift:61-122) and dq_rmsnorm +
// dq_rope (DirectGlueKernels.swift:14-75), queries and keys in one launch and
// one rounding at the end.
#include "core_kernels.hpp"
#include "imq_device.hpp"

namespace imq {
namespace {

constexpr int kThreads = 256;

// cos and sin of position * freq, times the amplitude.  An angle in radians
// loses its turns' fraction in 32 bits (position 2^20: 0.06 rad), so the
// product and the reduction to a quarter turn r in [-1/2, 1/2] are done in
// 64 bits; r itself then has an absolute error under 2^-25 in 32.
__device__ __forceinline__ float2 cos_sin(int position, double freq, float amplitude) {
  const double quarters = (double)position * (freq * 0.63661977236758134308);  // 2 / pi
  const double whole = rint(quarters);
  const float r = (float)(quarters - whole);
  float s, c;
  sincospif(0.5f * r, &s, &c);
  // whole modulo 4 (whole is up to 2^31 * freq: not always an int).
  const int n = (int)(whole - 4.0 * floor(whole * 0.25));
  if (n & 1) {
    const float t = c;
    c = -s;
    s = t;
  }
  if (n & 2) {
    c = -c;
    s = -s;
  }
  return make_float2(c * amplitude, s * amplitude);
}

__device__ __forceinline__ int axis_of(const RopeArgs& a, int pair) {
  return (pair >= a.section_end[0]) + (pair >= a.section_end[1]) + (pair >= a.section_end[2]);
}

template <int T>
__device__ __forceinline__ typename Elem<T>::S rounded(float v) {
  if constexpr (T == kF32) return v;
  else return (typename Elem<T>::S)(Elem<T>::pack2(v, v) & 0xFFFFu);
}

// Any dim, rotation, strides and alignment: a wave per row and head, a pair
// (then an element of the rest) per lane.
template <int T, bool kInterleaved>
__global__ __launch_bounds__(kThreads) void rope_kernel(RopeArgs a) {
  using S = typename Elem<T>::S;
  const int lane = threadIdx.x & 63;
  const int heads = a.g[0].heads + (a.groups > 1 ? a.g[1].heads : 0);
  const int64_t items = (int64_t)a.rows * heads;
  for (int64_t item = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6); item < items;
       item += (int64_t)gridDim.x * (kThreads / 64)) {
    const int row = (int)(item / heads);
    int h = (int)(item % heads);
    const int gi = h >= a.g[0].heads;
    const RopeGroup& g = a.g[gi];
    if (gi) h -= a.g[0].heads;
    const S* x = static_cast<const S*>(g.x) + row * g.x_row + h * g.x_head;
    S* y = static_cast<S*>(g.y) + row * g.y_row + h * g.y_head;
    float inv = 1.f;
    if (g.weight) {
      float acc = 0.f;
      for (int i = lane; i < a.dim; i += 64) {
        const float v = Elem<T>::param(x[i]);
        acc = __builtin_fmaf(v, v, acc);
      }
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) acc += __shfl_xor(acc, off, 64);
      inv = __frsqrt_rn(acc / (float)a.dim + a.eps);
    }
    const int half = a.rot / 2;
    for (int j = lane; j < half; j += 64) {
      const float2 cs = cos_sin(a.positions[(int64_t)row * a.axes + axis_of(a, j)], a.inv_freq[j],
                                a.amplitude);
      const int ia = kInterleaved ? 2 * j : j, ib = kInterleaved ? 2 * j + 1 : j + half;
      float u = Elem<T>::param(x[ia]), v = Elem<T>::param(x[ib]);
      if (g.weight) {
        u *= inv * g.weight[ia];
        v *= inv * g.weight[ib];
      }
      y[ia] = rounded<T>(u * cs.x - v * cs.y);
      y[ib] = rounded<T>(v * cs.x + u * cs.y);
    }
    for (int i = a.rot + lane; i < a.dim; i += 64) {
      const float v = Elem<T>::param(x[i]);
      y[i] = rounded<T>(g.weight ? v * (inv * g.weight[i]) : v);
    }
  }
}

template <int T>
hipError_t launch_t(const RopeArgs& a, bool interleaved, hipStream_t stream) {
  const int64_t heads = (int64_t)a.g[0].heads + (a.groups > 1 ? a.g[1].heads : 0);
  const int64_t blocks = (a.rows * heads + kThreads / 64 - 1) / (kThreads / 64);
  if (blocks == 0) return hipSuccess;
  const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : (1 << 20))), block(kThreads);
  if (interleaved)
    hipLaunchKernelGGL((rope_kernel<T, true>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((rope_kernel<T, false>), grid, block, 0, stream, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_rope(const RopeArgs& a, bool interleaved, int dtype, hipStream_t stream) {
  switch (dtype) {
    case kBf16: return launch_t<kBf16>(a, interleaved, stream);
    case kF16: return launch_t<kF16>(a, interleaved, stream);
    case kF32: return launch_t<kF32>(a, interleaved, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace imq
