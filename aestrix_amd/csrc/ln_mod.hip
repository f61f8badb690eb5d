// ln_mod.hip -- LayerNorm with the block's modulation into a qmm input.
//
// y[r][c] = T(((x[r][c] - mean) * rsqrt(var + eps) * (1 + scale[s][c]) + shift[s][c]) * post):
// the lnMod of a DiT block and of the head's norm_out in the shape of the
// reference's dd_ln_mod_prescale (Sources/ImarelloDirect/DirectDiTKernels.swift:16-59),
// a row picking its modulation s by an index.  Bound by HBM: x is read once into
// registers, y written once; the modulations stay in the caches.  4608 x 3072
// fp32 to f16: 15.8 us (5.4 TB/s, part of it cached; a 1 GiB copy reaches 5.18; a kernel that reads
// x three times 31.5); 1536 rows 8.0.
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
    const typename Elem<TX>::S* x, const float* __restrict__ shift,
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

// Four consecutive elements as floats.
template <int T>
__device__ __forceinline__ float4 load4(const typename Elem<T>::S* p) {
  if constexpr (T == kF32) {
    return *reinterpret_cast<const float4*>(p);
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    return make_float4(Elem<T>::param((uint16_t)(v.x & 0xFFFFu)), Elem<T>::param((uint16_t)(v.x >> 16)),
                       Elem<T>::param((uint16_t)(v.y & 0xFFFFu)), Elem<T>::param((uint16_t)(v.y >> 16)));
  }
}

// cols % 4 == 0: the row is read once and kept in registers, V float4 a lane,
// kWaves waves a row (1: four rows a workgroup, no barrier; 4: one row, whose
// loads are in flight together).
template <int TX, int TY, int kWaves, int V>
__global__ __launch_bounds__(kThreads) void ln_mod_vec_kernel(
    const typename Elem<TX>::S* x, const float* __restrict__ shift,
    const float* __restrict__ scale, const int32_t* __restrict__ sets, int n_sets,
    typename Elem<TY>::S* y, int rows, int cols, float eps, float post) {
  __shared__ float part[2][kThreads / 64];
  const int row = kWaves == 4 ? blockIdx.x : blockIdx.x * 4 + (threadIdx.x >> 6);
  if (kWaves == 1 && row >= rows) return;
  const int at = kWaves == 4 ? threadIdx.x : threadIdx.x & 63;
  const int n4 = cols >> 2;
  const typename Elem<TX>::S* xr = x + (size_t)row * cols;
  float4 v[V];
  float acc = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = at + i * 64 * kWaves;
    v[i] = c < n4 ? load4<TX>(xr + 4 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const int s = sets ? min(max(sets[row], 0), n_sets - 1) : 0;
#pragma unroll
  for (int i = 0; i < V; ++i) acc += (v[i].x + v[i].y) + (v[i].z + v[i].w);
  auto total = [&](float t, float* p) {
    if constexpr (kWaves == 4) return block_sum(t, p);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) t += __shfl_xor(t, off, 64);
    return t;
  };
  const float mean = total(acc, part[0]) / (float)cols;
  acc = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (at + i * 64 * kWaves < n4) {
      v[i].x -= mean, v[i].y -= mean, v[i].z -= mean, v[i].w -= mean;
      acc = __builtin_fmaf(v[i].x, v[i].x, acc);
      acc = __builtin_fmaf(v[i].y, v[i].y, acc);
      acc = __builtin_fmaf(v[i].z, v[i].z, acc);
      acc = __builtin_fmaf(v[i].w, v[i].w, acc);
    }
  const float inv = __frsqrt_rn(total(acc, part[1]) / (float)cols + eps);
  const float4* sc = reinterpret_cast<const float4*>(scale + (size_t)s * cols);
  const float4* sh = reinterpret_cast<const float4*>(shift + (size_t)s * cols);
  uint2* yr = reinterpret_cast<uint2*>(y + (size_t)row * cols);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = at + i * 64 * kWaves;
    if (c < n4) {
      const float4 a = sc[c], b = sh[c];
      yr[c] = make_uint2(Elem<TY>::pack2(__builtin_fmaf(v[i].x * inv, 1.f + a.x, b.x) * post,
                                         __builtin_fmaf(v[i].y * inv, 1.f + a.y, b.y) * post),
                         Elem<TY>::pack2(__builtin_fmaf(v[i].z * inv, 1.f + a.z, b.z) * post,
                                         __builtin_fmaf(v[i].w * inv, 1.f + a.w, b.w) * post));
    }
  }
}

template <int TX, int TY>
hipError_t launch_t(const void* x, const float* shift, const float* scale, const int32_t* sets,
                    int n_sets, void* y, int rows, int cols, float eps, float post,
                    hipStream_t stream) {
  const auto* xx = static_cast<const typename Elem<TX>::S*>(x);
  auto* yy = static_cast<typename Elem<TY>::S*>(y);
  const dim3 block(kThreads);
  const bool vec = cols % 4 == 0 && (uintptr_t)x % (4 * Elem<TX>::kBytes) == 0 &&
                   ((uintptr_t)shift | (uintptr_t)scale) % 16 == 0 && (uintptr_t)y % 8 == 0;
#define IMQ_LN_VEC(W, V)                                                                         \
  hipLaunchKernelGGL((ln_mod_vec_kernel<TX, TY, W, V>), dim3(W == 4 ? rows : (rows + 3) / 4), \
                     block, 0, stream, xx, shift, scale, sets, n_sets, yy, rows, cols, eps, post)
  // A wave a row for many short rows: 16384 x 512 12.6 us against 18.1, x 1024 22.8 /
  // 24.2, 4096 x 1024 6.9 / 7.2; but x 1280 26.8 / 27.5 and x 2048 43.0 / 37.7, 4608 x 3072
  // 21.6 / 19.6, 2048 x 1024 5.2 / 4.8 (in a captured graph over 500 MB of rows).
  if (vec && rows >= 4096 && cols <= 1024) {
    IMQ_LN_VEC(1, 4);
  } else if (vec && cols <= 8192) {
    if (cols <= 1024) IMQ_LN_VEC(4, 1);
    else if (cols <= 2048) IMQ_LN_VEC(4, 2);
    else if (cols <= 3072) IMQ_LN_VEC(4, 3);
    else if (cols <= 5120) IMQ_LN_VEC(4, 5);
    else IMQ_LN_VEC(4, 8);
  } else {
    hipLaunchKernelGGL((ln_mod_kernel<TX, TY>), dim3(rows), block, 0, stream, xx, shift, scale, sets,
                       n_sets, yy, cols, eps, post);
  }
#undef IMQ_LN_VEC
  return hipGetLastError();
}

}  // namespace

hipError_t launch_ln_mod(const void* x, int x_dtype, const float* shift, const float* scale,
                         const int32_t* sets, int n_sets, void* y, int y_dtype, int rows, int cols,
                         float eps, float post, hipStream_t stream) {
  constexpr int kMost = 1 << 23;  // rows of a launch: its threads stay under 2^32
  if (rows <= 0) return hipSuccess;
  if (rows > kMost) {
    for (int64_t r = 0; r < rows; r += kMost) {
      const size_t at = (size_t)r * cols;
      const hipError_t e = launch_ln_mod(
          static_cast<const char*>(x) + at * (x_dtype == kF32 ? 4 : 2), x_dtype, shift, scale,
          sets ? sets + r : nullptr, n_sets, static_cast<char*>(y) + at * 2, y_dtype,
          (int)(rows - r < kMost ? rows - r : kMost), cols, eps, post, stream);
      if (e != hipSuccess) return e;
    }
    return hipSuccess;
  }
#define IMQ_LN_MOD(TX, TY) \
  return launch_t<TX, TY>(x, shift, scale, sets, n_sets, y, rows, cols, eps, post, stream)
  if (x_dtype == kF32 && y_dtype == kBf16) IMQ_LN_MOD(kF32, kBf16);
  if (x_dtype == kF32 && y_dtype == kF16) IMQ_LN_MOD(kF32, kF16);
  if (x_dtype == kBf16 && y_dtype == kBf16) IMQ_LN_MOD(kBf16, kBf16);
  if (x_dtype == kF16 && y_dtype == kF16) IMQ_LN_MOD(kF16, kF16);
#undef IMQ_LN_MOD
  return hipErrorInvalidValue;
}

}  // namespace imq
