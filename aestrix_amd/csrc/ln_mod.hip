// ln_mod.hip -- LayerNorm with the block's modulation into a qmm input.
//
// y[r][c] = T(((x[r][c] - mean) * rsqrt(var + eps) * (1 + scale[s][c]) + shift[s][c]) * post):
// the lnMod of a DiT block and of the head's norm_out in the shape of the
// reference's dd_ln_mod_prescale (Sources/ImarelloDirect/DirectDiTKernels.swift:16-59),
// a row picking its modulation s by an index.
#include "core_kernels.hpp"
#include "imq_device.hpp"

namespace imq {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float block_sum(float v, float* part) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) t += part[i];
  return t;
}

// Any cols and alignment; the row is read three times (from the cache after
// the first).  The variance is that of the differences from the mean: sums of
// squares would cancel where a row's mean is large against its spread.
template <int TX, int TY>
__global__ __launch_bounds__(kThreads) void ln_mod_kernel(
    const typename Elem<TX>::S* __restrict__ x, const float* __restrict__ shift,
    const float* __restrict__ scale, const int32_t* __restrict__ sets, int n_sets,
    typename Elem<TY>::S* y, int cols, float eps, float post) {
  __shared__ float part[2][kThreads / 64];
  const typename Elem<TX>::S* xr = x + (size_t)blockIdx.x * cols;
  float acc = 0.f;
  for (int c = threadIdx.x; c < cols; c += kThreads) acc += Elem<TX>::param(xr[c]);
  const float mean = block_sum(acc, part[0]) / (float)cols;
  acc = 0.f;
  for (int c = threadIdx.x; c < cols; c += kThreads) {
    const float d = Elem<TX>::param(xr[c]) - mean;
    acc = __builtin_fmaf(d, d, acc);
  }
  const float inv = __frsqrt_rn(block_sum(acc, part[1]) / (float)cols + eps);
  const int s = sets ? min(max(sets[blockIdx.x], 0), n_sets - 1) : 0;
  const float* sc = scale + (size_t)s * cols;
  const float* sh = shift + (size_t)s * cols;
  typename Elem<TY>::S* yr = y + (size_t)blockIdx.x * cols;
  for (int c = threadIdx.x; c < cols; c += kThreads) {
    const float n = (Elem<TX>::param(xr[c]) - mean) * inv;
    const float v = __builtin_fmaf(n, 1.f + sc[c], sh[c]) * post;
    yr[c] = (typename Elem<TY>::S)(Elem<TY>::pack2(v, v) & 0xFFFFu);
  }
}

}  // namespace

hipError_t launch_ln_mod(const void* x, int x_dtype, const float* shift, const float* scale,
                         const int32_t* sets, int n_sets, void* y, int y_dtype, int rows, int cols,
                         float eps, float post, hipStream_t stream) {
  if (rows <= 0) return hipSuccess;
  const dim3 grid(rows), block(kThreads);
  auto* yy = static_cast<uint16_t*>(y);
#define IMQ_LN_MOD(TX, TY)                                                                      \
  hipLaunchKernelGGL((ln_mod_kernel<TX, TY>), grid, block, 0, stream,                           \
                     static_cast<const Elem<TX>::S*>(x), shift, scale, sets, n_sets, yy, cols, \
                     eps, post)
  if (x_dtype == kF32 && y_dtype == kBf16) IMQ_LN_MOD(kF32, kBf16);
  else if (x_dtype == kF32 && y_dtype == kF16) IMQ_LN_MOD(kF32, kF16);
  else if (x_dtype == kBf16 && y_dtype == kBf16) IMQ_LN_MOD(kBf16, kBf16);
  else if (x_dtype == kF16 && y_dtype == kF16) IMQ_LN_MOD(kF16, kF16);
  else return hipErrorInvalidValue;
#undef IMQ_LN_MOD
  return hipGetLastError();
}

}  // namespace imq
