// rope.hip -- per-head RMSNorm and rotary positions of the query and key heads.
//
// y = turn(x * rsqrt(mean(x^2) + eps) * w) by angle_j = position * inv_freq[j]:
// the reference's dd_rmsnorm_pitched + dd_rope_interleaved
// (Sources/ImarelloDirect/DirectDiTKernels.swift:61-122) and dq_rmsnorm +
// dq_rope (DirectGlueKernels.swift:14-75), queries and keys in one launch and
// one rounding at the end.  Bound by HBM: a head is read and written once.  4608
// rows of 48 heads of 128 in f16, normed: 22-25 us (a 1 GiB copy's rate: 21.8;
// a wave a head and a pair a lane, below: 100); 16001 rows of 40 heads in bf16, half of
// each turned: 65 us (5.0 TB/s; 245); 4 rows: 4.4 us, a launch and four round trips.
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

// 8 consecutive elements: 16 bytes (two pieces of 16 in f32).
template <int T>
struct Piece8 {
  uint4 v[T == kF32 ? 2 : 1];
};

template <int T>
__device__ __forceinline__ Piece8<T> load8(const typename Elem<T>::S* p) {
  Piece8<T> r;
  const uint4* q = reinterpret_cast<const uint4*>(p);
  r.v[0] = q[0];
  if constexpr (T == kF32) r.v[1] = q[1];
  return r;
}

template <int T>
__device__ __forceinline__ void unpack8(const Piece8<T>& p, float f[8]) {
  const uint32_t w[4] = {p.v[0].x, p.v[0].y, p.v[0].z, p.v[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (T == kF32) {
      const uint32_t w1[4] = {p.v[1].x, p.v[1].y, p.v[1].z, p.v[1].w};
      f[i] = __uint_as_float(w[i]);
      f[4 + i] = __uint_as_float(w1[i]);
    } else {
      f[2 * i] = Elem<T>::param((uint16_t)(w[i] & 0xFFFFu));
      f[2 * i + 1] = Elem<T>::param((uint16_t)(w[i] >> 16));
    }
  }
}

template <int T>
__device__ __forceinline__ void store8(typename Elem<T>::S* p, const float f[8]) {
  uint4* q = reinterpret_cast<uint4*>(p);
  if constexpr (T == kF32) {
    q[0] = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                      __float_as_uint(f[3]));
    q[1] = make_uint4(__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]),
                      __float_as_uint(f[7]));
  } else {
    q[0] = make_uint4(Elem<T>::pack2(f[0], f[1]), Elem<T>::pack2(f[2], f[3]),
                      Elem<T>::pack2(f[4], f[5]), Elem<T>::pack2(f[6], f[7]));
  }
}

constexpr int kMaxVecDim = 512;
constexpr int kBatch = 3;  // head groups a wave holds at once: their loads are in flight together

// The vector form: a lane holds 16 elements of a head (the two 8-element sides
// of 8 pairs in the half layout, 16 consecutive ones interleaved or not
// turned), 2^lanes_log2 lanes a head.  The angles of a row are computed once,
// a pair per thread, and every lane keeps the cos and sin of its 8 pairs in
// registers over all heads: the angle in fp64 and its sine are some 60
// instructions, against 16 elements of a head.  kRows rows a workgroup: 4, a
// wave each (a row's heads then share one set of angles), where there are many;
// 1, its heads over the four waves, where there are few.
template <int T, bool kInterleaved, int kRows>
__global__ __launch_bounds__(kThreads) void rope_vec_kernel(RopeArgs a, int lanes_log2) {
  using S = typename Elem<T>::S;
  __shared__ float2 cs[kRows][kMaxVecDim / 2];
  const int half = a.rot / 2;
  const int row0 = blockIdx.x * kRows;
  for (int i = threadIdx.x; i < kRows * half; i += kThreads) {
    const int r = i / half, j = i % half;
    if (row0 + r < a.rows)
      cs[r][j] = cos_sin(a.positions[(int64_t)(row0 + r) * a.axes + axis_of(a, j)], a.inv_freq[j],
                         a.amplitude);
  }
  __syncthreads();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row = row0 + (kRows == 4 ? wave : 0);
  if (row >= a.rows) return;
  const int unit = lane & ((1 << lanes_log2) - 1), sub = lane >> lanes_log2;
  const int per = 64 >> lanes_log2;  // heads of a wave's group
  const bool turned = 16 * unit < a.rot, used = 16 * unit < a.dim;
  const int e0 = !kInterleaved && turned ? 8 * unit : 16 * unit;
  const int e1 = !kInterleaved && turned ? 8 * unit + half : 16 * unit + 8;
  float2 t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    t[i] = turned ? cs[kRows == 4 ? wave : 0][8 * unit + i] : make_float2(1.f, 0.f);
#pragma unroll 1
  for (int gi = 0; gi < a.groups; ++gi) {
    const RopeGroup g = a.g[gi];
    const S* x = static_cast<const S*>(g.x) + row * g.x_row;
    S* y = static_cast<S*>(g.y) + row * g.y_row;
    float w0[8], w1[8];
    if (g.weight && used) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 u = *reinterpret_cast<const float4*>(g.weight + e0 + 4 * i);
        const float4 v = *reinterpret_cast<const float4*>(g.weight + e1 + 4 * i);
        w0[4 * i] = u.x, w0[4 * i + 1] = u.y, w0[4 * i + 2] = u.z, w0[4 * i + 3] = u.w;
        w1[4 * i] = v.x, w1[4 * i + 1] = v.y, w1[4 * i + 2] = v.z, w1[4 * i + 3] = v.w;
      }
    }
    const int step = kRows == 4 ? per : 4 * per;
    for (int h0 = (kRows == 4 ? 0 : wave * per) + sub; h0 - sub < g.heads; h0 += kBatch * step) {
      Piece8<T> p0[kBatch], p1[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int h = h0 + b * step;
        if (used && h < g.heads) {
          p0[b] = load8<T>(x + h * g.x_head + e0);
          p1[b] = load8<T>(x + h * g.x_head + e1);
        } else {
          p0[b] = p1[b] = Piece8<T>{};
        }
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int h = h0 + b * step;
        if (h - sub >= g.heads) break;  // for the whole wave
        float u[8], v[8];
        unpack8<T>(p0[b], u);
        unpack8<T>(p1[b], v);
        if (g.weight) {
          float acc = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            acc = __builtin_fmaf(u[i], u[i], acc);
            acc = __builtin_fmaf(v[i], v[i], acc);
          }
          for (int off = (1 << lanes_log2) >> 1; off > 0; off >>= 1) acc += __shfl_xor(acc, off, 64);
          const float inv = __frsqrt_rn(acc / (float)a.dim + a.eps);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            u[i] *= inv * w0[i];
            v[i] *= inv * w1[i];
          }
        }
        if (turned) {
          if constexpr (kInterleaved) {
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
              const float2 c0 = t[i / 2], c1 = t[4 + i / 2];
              const float u0 = u[i], u1 = u[i + 1], v0 = v[i], v1 = v[i + 1];
              u[i] = u0 * c0.x - u1 * c0.y;
              u[i + 1] = u1 * c0.x + u0 * c0.y;
              v[i] = v0 * c1.x - v1 * c1.y;
              v[i + 1] = v1 * c1.x + v0 * c1.y;
            }
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float u0 = u[i], v0 = v[i];
              u[i] = u0 * t[i].x - v0 * t[i].y;
              v[i] = v0 * t[i].x + u0 * t[i].y;
            }
          }
        }
        if (used && h < g.heads) {
          store8<T>(y + h * g.y_head + e0, u);
          store8<T>(y + h * g.y_head + e1, v);
        }
      }
    }
  }
}

bool vec_fits(const RopeArgs& a, int es) {
  if (a.dim % 16 != 0 || a.rot % 16 != 0 || a.dim > kMaxVecDim) return false;
  for (int i = 0; i < a.groups; ++i) {
    const RopeGroup& g = a.g[i];
    if (((uintptr_t)g.x | (uintptr_t)g.y | (uintptr_t)g.weight) % 16 != 0) return false;
    if ((g.x_row | g.x_head | g.y_row | g.y_head) * es % 16 != 0) return false;
  }
  return true;
}

template <int T>
hipError_t launch_t(const RopeArgs& a, bool interleaved, hipStream_t stream) {
  const int64_t heads = (int64_t)a.g[0].heads + (a.groups > 1 ? a.g[1].heads : 0);
  const int64_t blocks = (a.rows * heads + kThreads / 64 - 1) / (kThreads / 64);
  if (blocks == 0) return hipSuccess;
  const dim3 block(kThreads);
  if (vec_fits(a, Elem<T>::kBytes)) {
    int log2 = 0;
    while ((16 << log2) < a.dim) ++log2;
    // Many rows against a row's width: 4096 rows of 5 heads of 128 6.3 us against
    // 11.2, 2048 of 20 8.1 / 9.7, 3072 of 48 15.3 / 15.9; but 1024 of 48 9.8 / 7.7,
    // 2048 of 48 12.5 / 11.9, 2048 of 32 of 256 16.7 / 14.3; 16384 rows level.
    const bool many = 5 * (int64_t)a.rows >= 2 * heads * a.dim;
    const dim3 grid((unsigned)(many ? (a.rows + 3) / 4 : a.rows));
    if (interleaved && many)
      hipLaunchKernelGGL((rope_vec_kernel<T, true, 4>), grid, block, 0, stream, a, log2);
    else if (interleaved)
      hipLaunchKernelGGL((rope_vec_kernel<T, true, 1>), grid, block, 0, stream, a, log2);
    else if (many)
      hipLaunchKernelGGL((rope_vec_kernel<T, false, 4>), grid, block, 0, stream, a, log2);
    else
      hipLaunchKernelGGL((rope_vec_kernel<T, false, 1>), grid, block, 0, stream, a, log2);
    return hipGetLastError();
  }
  const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)));
  if (interleaved)
    hipLaunchKernelGGL((rope_kernel<T, true>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((rope_kernel<T, false>), grid, block, 0, stream, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_rope(const RopeArgs& a, bool interleaved, int dtype, hipStream_t stream) {
  constexpr int kMost = 1 << 23;  // rows of a launch: its threads stay under 2^32
  if (a.rows > kMost) {
    const int64_t es = dtype == kF32 ? 4 : 2;
    for (int64_t r = 0; r < a.rows; r += kMost) {
      RopeArgs part = a;
      part.rows = (int)(a.rows - r < kMost ? a.rows - r : kMost);
      if (a.positions) part.positions = a.positions + r * a.axes;
      for (int i = 0; i < a.groups; ++i) {
        part.g[i].x = static_cast<const char*>(a.g[i].x) + r * a.g[i].x_row * es;
        part.g[i].y = static_cast<char*>(a.g[i].y) + r * a.g[i].y_row * es;
      }
      const hipError_t e = launch_rope(part, interleaved, dtype, stream);
      if (e != hipSuccess) return e;
    }
    return hipSuccess;
  }
  switch (dtype) {
    case kBf16: return launch_t<kBf16>(a, interleaved, stream);
    case kF16: return launch_t<kF16>(a, interleaved, stream);
    case kF32: return launch_t<kF32>(a, interleaved, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace imq
