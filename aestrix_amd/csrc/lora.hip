// lora.hip -- the products of adapters beside a projection that stand outside its kernels: u =
// scale * A x, a row's adapter's, and the join of the projection's partial sums with B u
// (include/imq_lora.h).
#include <algorithm>

#include "lora_device.hpp"

namespace imq {
namespace {

// ---- u

// The rows of a tile by what adapters they name; a lane's row is r32 (in both halves).
struct LoraRows {
  int id;     // of this lane's row, -1: none
  LoraAt at;  // its adapter's, looked up for all rows together

  __device__ __forceinline__ LoraRows(const LoraArgs& l, int row, int m) {
    id = row < m ? lora_of(l, row) : -1;
    at = lora_at(l, max(id, 0));
  }
  // The j-th adapter (from 0) that they name, in the order of their first rows, and its rows; -1
  // where there are fewer.
  __device__ __forceinline__ int nth(int j, uint32_t& rows, LoraAt& to) const {
    uint32_t left = (uint32_t)__builtin_amdgcn_ballot_w64(id >= 0);
    while (left) {
      const int lead = __builtin_ctz(left), i = __builtin_amdgcn_readlane(id, lead);
      rows = (uint32_t)__builtin_amdgcn_ballot_w64(id == i);
      if (j-- == 0) {
        to = LoraAt{__builtin_amdgcn_readlane(at.row, lead), __builtin_amdgcn_readlane(at.rank, lead)};
        return i;
      }
      left &= ~rows;
    }
    return -1;
  }
};

constexpr int kDotWaves = 4;
template <int T, int kAhead>
__global__ __launch_bounds__(kDotWaves * 64) void lora_dot_kernel(LoraArgs l, const uint16_t* x, int k, int m) {
  lora_dot<T, kAhead>(l, x, k, m, blockIdx.x * kDotWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
}

// More rows.  A workgroup: 32 of them against 32 ranks (blockIdx.y) of the adapters that they
// name, every second one (blockIdx.z).  Its eight waves take K in turn, 64 at a time, from buffers
// of their own: whole 128-byte lines of x's and A's rows straight to LDS (operands loaded straight
// to registers touch 32 bytes of a line each, and 16 such waves took 35 us of 4608 rows of 2560
// against one adapter of rank 64, this 14), the next piece on its way while one is multiplied.
// 16-byte pieces are swizzled by the row at their source, so that the operand reads touch every
// bank evenly.  The waves' sums are added through LDS.  Bound by the latency of the loads, of
// `which` and `first` before them: 4000 rows of 2560 in runs of 100 of rank 16 12 us.
constexpr int kShrinkWaves = 8;
struct ShrinkBuf {
  uint4 x[32 * 8], a[32 * 8];
};
template <int T>
__global__ __launch_bounds__(kShrinkWaves * 64) void lora_shrink_kernel(LoraArgs l, const uint16_t* x,
                                                                       int k, int m) {
  __shared__ union {
    ShrinkBuf buf[kShrinkWaves][2];
    float sums[kShrinkWaves][32 * 32];
  } lds;
  const int lane = threadIdx.x & 63, r32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tile = blockIdx.x, r0 = blockIdx.y * 32;
  const int pieces = k / 64;
  const uint32_t kb = (uint32_t)k * 2;
  // This lane's 16 bytes of the rows 8 s + lane / 8; grouped rows stand anywhere in x, which is
  // under 2^31 bytes then.
  const __amdgpu_buffer_rsrc_t xr =
      l.order ? make_rsrc(x, (uint32_t)m * kb)
              : make_rsrc(x + (size_t)tile * 32 * k, (uint32_t)min(32, m - tile * 32) * kb);
  uint32_t x_off[4], a_off[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const uint32_t r = s * 8 + lane / 8, c = ((lane ^ r) & 7) * 16;
    a_off[s] = r * kb + c;
    x_off[s] = l.order ? (uint32_t)l.order[min(tile * 32 + (int)r, m - 1)] * kb + c : a_off[s];
  }
  auto load_x = [&](int p, int set) {
#pragma unroll
    for (int s = 0; s < 4; ++s)
      load_lds16(xr, x_off[s], (uint32_t)min(p, pieces - 1) * 128, lds.buf[wave][set].x + s * 64);
  };
  // The first adapter's x, before it is known which that is.
  load_x(wave, 0);
  const LoraRows of_tile(l, tile * 32 + r32, m);
  uint32_t rows;
  LoraAt at;
  bool ahead = true;
  for (int j = blockIdx.z;; j += gridDim.z) {
    const int i = of_tile.nth(j, rows, at);
    if (i < 0) break;
    if (r0 >= at.rank) continue;
    // (Ranks past the last are zeros.)
    const __amdgpu_buffer_rsrc_t ar =
        make_rsrc(l.a + (size_t)(at.row + r0) * k, (uint32_t)min(32, at.rank - r0) * kb);
    f32x16_t c;
#pragma unroll
    for (int e = 0; e < 16; ++e) c[e] = 0.f;
    // (Past the last piece it is loaded again, so that the counts of loads in flight hold.)
    auto load_a = [&](int p, int set) {
#pragma unroll
      for (int s = 0; s < 4; ++s)
        load_lds16(ar, a_off[s], (uint32_t)min(p, pieces - 1) * 128, lds.buf[wave][set].a + s * 64);
    };
    if (!ahead) load_x(wave, 0);
    ahead = false;
    load_a(wave, 0);
    int set = 0;
    for (int p = wave; p < pieces; p += kShrinkWaves, set ^= 1) {
      __builtin_amdgcn_sched_barrier(0);
      load_x(p + kShrinkWaves, set ^ 1);
      load_a(p + kShrinkWaves, set ^ 1);
      __builtin_amdgcn_sched_barrier(0);
      IMQ_WAIT_VMCNT(8);  // this piece has landed
      __builtin_amdgcn_sched_barrier(0);
      const ShrinkBuf& from = lds.buf[wave][set];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int slot = r32 * 8 + ((2 * s + h) ^ (r32 & 7));
        c = lora_mfma<T>(__builtin_bit_cast(u32x4_t, from.x[slot]), __builtin_bit_cast(u32x4_t, from.a[slot]), c);
      }
      __builtin_amdgcn_sched_barrier(0);
      IMQ_WAIT_LGKM_0();  // and has been read
    }
    const int rank = r0 + (threadIdx.x & 31);  // of this thread's sums below
    const float scale = lora_scale(l, i, at.row + min(rank, at.rank - 1));
    __builtin_amdgcn_sched_barrier(0);
    IMQ_WAIT_VMCNT(0);
    __syncthreads();  // every wave's pieces have landed and been read
#pragma unroll
    for (int e = 0; e < 16; ++e) lds.sums[wave][(8 * (e >> 2) + 4 * h + (e & 3)) * 32 + r32] = c[e];
    __syncthreads();
#pragma unroll
    for (int o = threadIdx.x; o < 32 * 32; o += kShrinkWaves * 64) {
      const int of = o >> 5;
      float u = 0.f;
#pragma unroll
      for (int v = 0; v < kShrinkWaves; ++v) u += lds.sums[v][o];
      if ((rows >> of & 1u) && rank < at.rank) lora_put<T>(l, tile * 32 + of, rank, u * scale);
    }
    __syncthreads();  // the sums have been read
  }
  IMQ_WAIT_VMCNT(0);  // x of no adapter, before the workgroup's LDS is another's
}

// ---- the order of the rows

// One workgroup: each of its 16 waves counts the rows of a stretch by adapter, the counts are
// added up over adapters and waves, and each wave gives its rows their places, 64 at a time, in
// their order.  The adapters of kOrderKeep rows stay in LDS in between.  Loops are kept rolled: of
// code that runs once, fetching it is what takes the time (4.9 us of 777 rows, 7.7 of 4608).  More adapters
// than kOrderBins - 1: the rows stay as they are.
constexpr int kOrderWaves = 16, kOrderBins = 1024, kOrderKeep = 16384;
__global__ __launch_bounds__(kOrderWaves * 64) void lora_order_kernel(LoraArgs l, int32_t* order,
                                                                     int32_t* which_at, int m) {
  __shared__ int at[kOrderWaves][kOrderBins];
  __shared__ int sums[kOrderBins];
  __shared__ uint16_t kept[kOrderKeep];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int bins = l.count + 1;  // the last one: no adapter
  if (bins > kOrderBins) {
    for (int r = t; r < m; r += kOrderWaves * 64) {
      order[r] = r;
      which_at[r] = lora_of(l, r);
    }
    return;
  }
  auto load = [&](int r) {
    const int i = lora_of(l, r);
    return i < 0 ? l.count : i;
  };
  const int few = min(m, kOrderKeep);
  for (int r = t * 4; r < few; r += kOrderWaves * 256) {  // four at a time, whatever the alignment
    int v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = load(min(r + e, few - 1));
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (r + e < few) kept[r + e] = (uint16_t)v[e];
  }
  if (t < bins)
#pragma unroll 1
    for (int w = 0; w < kOrderWaves; ++w) at[w][t] = 0;
  __syncthreads();
  const int per = ((m + kOrderWaves - 1) / kOrderWaves + 63) / 64 * 64;
  const int begin = min(wave * per, m), end = min(begin + per, m);
  auto bin = [&](int r) { return r < kOrderKeep ? (int)kept[r] : load(r); };
  // The rows of [begin, end) 64 at a time, by the bins that they have; a bin's count or place is its
  // wave's alone.  (Atomics of 64 lanes on one bin took 4 us of 4000 rows' 9.)
  auto each = [&](auto visit) {
#pragma unroll 1
    for (int r0 = begin; r0 < end; r0 += 64) {
      const int r = r0 + lane, b = r < end ? bin(r) : -1;
      uint64_t left = __builtin_amdgcn_ballot_w64(b >= 0);
      while (left) {
        const int i = __builtin_amdgcn_readlane(b, __builtin_ctzll(left));
        const uint64_t rows = __builtin_amdgcn_ballot_w64(b == i);
        left &= ~rows;
        const int from = at[wave][i];
        __builtin_amdgcn_wave_barrier();
        visit(r, i, rows, from, b == i);
        if (lane == 0) at[wave][i] = from + __builtin_popcountll(rows);
        __builtin_amdgcn_wave_barrier();
      }
    }
  };
  each([](int, int, uint64_t, int, bool) {});
  __syncthreads();
  // Of every bin its rows, then over the bins (a scan by doubling steps).
  int mine = 0;
  if (t < bins)
#pragma unroll 1
    for (int w = 0; w < kOrderWaves; ++w) mine += at[w][t];
  sums[t] = mine;
  __syncthreads();
#pragma unroll 1
  for (int step = 1; step < bins; step *= 2) {
    const int v = t >= step ? sums[t - step] : 0;
    __syncthreads();
    sums[t] += v;
    __syncthreads();
  }
  if (t < bins) {
    int from = sums[t] - mine;
#pragma unroll 1
    for (int w = 0; w < kOrderWaves; ++w) {
      const int n = at[w][t];
      at[w][t] = from;
      from += n;
    }
  }
  __syncthreads();
  each([&](int r, int i, uint64_t rows, int from, bool mine) {
    if (!mine) return;
    const int to = from + __builtin_popcountll(rows & (((uint64_t)1 << lane) - 1));
    order[to] = r;
    which_at[to] = i < l.count ? i : -1;
  });
}

// ---- the join

// A thread an output, one row a workgroup, B's row against u in 32 bits.  Bound by the latency of
// `which`, `first` and B, one after the other, the ranges' sums on the way meanwhile ([16 x 6144] with
// 16 adapters of rank 16 4.5 us), and of many rows or ranks by reading B's rows, each for its row alone.
template <int T>
__global__ __launch_bounds__(256) void lora_join_few_kernel(LoraArgs l, const float* part, int splits,
                                                            uint16_t* y, int n, int m) {
  __shared__ float us[kLoraMaxRank];
  const int row = blockIdx.y, t = threadIdx.x, col = blockIdx.x * 256 + t;
  const float* from = part + (size_t)row * n + min(col, n - 1);
  const size_t range = (size_t)m * n;
  constexpr int kAhead = 8;
  float v[kAhead];
#pragma unroll
  for (int e = 0; e < kAhead; ++e) v[e] = from[min(e, splits - 1) * range];
  const int i = lora_of(l, row);
  float dot = 0.f;
  if (i >= 0) {
    const LoraAt at = lora_at(l, i);
    const u32x4_t* b = reinterpret_cast<const u32x4_t*>(l.b + (size_t)at.row * n + (size_t)min(col, n - 1) * at.rank);
    if (t < at.rank) {
      const uint16_t* u = l.u + (((size_t)(row / 32) * (l.max_rank / 16) + t / 16) * 2 * 64 + row % 32 +
                                 32 * (t >> 3 & 1)) * 8 + (t & 7);
      us[t] = staged_value<T>(u[0]) + staged_value<T>(u[64 * 8]);
    }
    __syncthreads();
#pragma unroll 2
    for (int r = 0; r < at.rank / 16; ++r) {
      const u32x4_t w[2] = {b[2 * r], b[2 * r + 1]};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        dot = __builtin_fmaf(staged_value<T>(w[e / 4][e % 4] & 0xFFFFu), us[16 * r + 2 * e], dot);
        dot = __builtin_fmaf(staged_value<T>(w[e / 4][e % 4] >> 16), us[16 * r + 2 * e + 1], dot);
      }
    }
  }
  float sum = v[0];
#pragma unroll
  for (int e = 1; e < kAhead; ++e) sum += e < splits ? v[e] : 0.f;
  for (int sp = kAhead; sp < splits; ++sp) sum += from[sp * range];
  if (col < n) y[(size_t)row * n + col] = Elem<T>::out(sum + dot);
}

// Long rows of B for many rows of y.  A workgroup: 32 rows and 32 columns of y.  Its 16 waves take the adapters of the rows in
// turn; each writes its rows' products to LDS (a row has one adapter), where the ranges' sums
// are added to them in order.  Bound by the latency of what a wave loads for an adapter; the
// ranges' sums are on the way meanwhile.  64 rows of N = 6144 with one adapter of rank 256 33 us a call with
// this join, 45 with the other.
constexpr int kJoinWaves = 16;  // a thread an output
template <int T>
__global__ __launch_bounds__(kJoinWaves * 64, 8) void lora_join_kernel(LoraArgs l, const float* part, int splits,
                                                                   uint16_t* y, int n, int m) {
  __shared__ float add[32 * 32];
  const int lane = threadIdx.x & 63, r32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * 32, tile = blockIdx.y;
  const int col = n0 + (int)(threadIdx.x & 31), of = threadIdx.x >> 5;  // of this thread's output
  const float* from = part + (size_t)min(tile * 32 + of, m - 1) * n + min(col, n - 1);
  const size_t range = (size_t)m * n;
  // The first ranges' sums are on their way while the adapters' products are made.
  constexpr int kAhead = 4;
  float v[kAhead];
#pragma unroll
  for (int e = 0; e < kAhead; ++e) v[e] = from[min(e, splits - 1) * range];
  const LoraRows of_tile(l, tile * 32 + r32, m);
  add[threadIdx.x] = 0.f;
  __syncthreads();
  uint32_t rows;
  LoraAt at;
  for (int j = wave; of_tile.nth(j, rows, at) >= 0; j += kJoinWaves) {
    const f32x16_t c = lora_product<T>(l, at, tile, n0, n);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int r = 8 * (e >> 2) + 4 * h + (e & 3);
      if (rows >> r & 1u) add[r * 32 + r32] = c[e];
    }
  }
  float sum = v[0];
#pragma unroll
  for (int e = 1; e < kAhead; ++e) sum += e < splits ? v[e] : 0.f;
  for (int sp = kAhead; sp < splits; ++sp) sum += from[sp * range];
  __syncthreads();
  if (tile * 32 + of < m && col < n)
    y[(size_t)(tile * 32 + of) * n + col] = Elem<T>::out(sum + add[threadIdx.x]);
}

}  // namespace

hipError_t launch_lora_order(const LoraArgs& l, int32_t* order, int32_t* which_at, int m, hipStream_t stream) {
  hipLaunchKernelGGL(lora_order_kernel, dim3(1), dim3(kOrderWaves * 64), 0, stream, l, order, which_at, m);
  return hipGetLastError();
}

// By the times of both in us.  That one reads A's and x's
// rows out of the caches, some 30 TB/s, whatever adapters the rows name; a tile of 32 rows
// takes its adapters two at a time, as many as it may have (all, or after grouping its share), 6 us
// of K = 2560 and 12 of 9728 each turn.  160 rows of 24 adapters of rank 16 in turn against K = 9728
// and N = 2560 30.8 us so, 168 by tiles; 64 rows of one adapter of rank 256 and K = 2560 44.7 and
// 41.4; 512 rows of 32 adapters of rank 64, grouped, 74.8 and 64.4.
bool lora_by_rows(int count, int max_rank, bool grouped, int k, int m) {
  const double rows_us = 2 + 4. * m * max_rank * k / 30e6;
  const int most = std::min(std::min(count, m), grouped ? 1 + (int)((int64_t)count * 32 / m) : 32);
  return rows_us <= (most + 1) / 2 * (3.5 + k * 0.0009) && (int64_t)m * max_rank < 1 << 24;
}

double lora_join_few_us(int n, int m, int max_rank) { return 2. * m * n * max_rank / 10e6; }
double lora_join_tiles_us(int n, int m, int count, int max_rank) {
  const int most = std::min(std::min(count, m), 32);
  const double rows = (m + 31) / 32;
  return 1.5 + (1.2 + 0.27 * most) * ((n + 31) / 32) * rows / 256 + 2. * rows * most * n * max_rank / 3e6;
}

bool lora_join_few(int n, int m, int count, int max_rank) {
  return m <= 65535 && lora_join_few_us(n, m, max_rank) <= lora_join_tiles_us(n, m, count, max_rank);
}

hipError_t launch_lora_shrink(const LoraArgs& l, const void* x, int k, int m, int dtype,
                              hipStream_t stream) {
  const auto* xx = static_cast<const uint16_t*>(x);
  if (lora_by_rows(l.count, l.max_rank, l.order != nullptr, k, m)) {
    const dim3 grid((unsigned)((m * l.max_rank + kDotWaves - 1) / kDotWaves)), block(kDotWaves * 64);
    // Rows of more than 8 KB: 20 pieces at a time, of which shorter rows would have too few.
    if (k > 4096) {
      if (dtype == kBf16)
        hipLaunchKernelGGL((lora_dot_kernel<kBf16, 20>), grid, block, 0, stream, l, xx, k, m);
      else
        hipLaunchKernelGGL((lora_dot_kernel<kF16, 20>), grid, block, 0, stream, l, xx, k, m);
    } else {
      if (dtype == kBf16)
        hipLaunchKernelGGL((lora_dot_kernel<kBf16, 8>), grid, block, 0, stream, l, xx, k, m);
      else
        hipLaunchKernelGGL((lora_dot_kernel<kF16, 8>), grid, block, 0, stream, l, xx, k, m);
    }
    return hipGetLastError();
  }
  const dim3 grid((unsigned)((m + 31) / 32), (unsigned)((l.max_rank + 31) / 32), l.count > 1 ? 2 : 1),
      block(kShrinkWaves * 64);
  if (dtype == kBf16)
    hipLaunchKernelGGL((lora_shrink_kernel<kBf16>), grid, block, 0, stream, l, xx, k, m);
  else
    hipLaunchKernelGGL((lora_shrink_kernel<kF16>), grid, block, 0, stream, l, xx, k, m);
  return hipGetLastError();
}

hipError_t launch_lora_join(const LoraArgs& l, const float* part, int splits, void* y, int n, int m,
                            int dtype, hipStream_t stream) {
  auto* yy = static_cast<uint16_t*>(y);
  if (lora_join_few(n, m, l.count, l.max_rank)) {
    const dim3 grid((unsigned)((n + 255) / 256), (unsigned)m);
    if (dtype == kBf16)
      hipLaunchKernelGGL((lora_join_few_kernel<kBf16>), grid, dim3(256), 0, stream, l, part, splits, yy, n, m);
    else
      hipLaunchKernelGGL((lora_join_few_kernel<kF16>), grid, dim3(256), 0, stream, l, part, splits, yy, n, m);
    return hipGetLastError();
  }
  const dim3 grid((unsigned)((n + 31) / 32), (unsigned)((m + 31) / 32)), block(kJoinWaves * 64);
  if (dtype == kBf16)
    hipLaunchKernelGGL((lora_join_kernel<kBf16>), grid, block, 0, stream, l, part, splits, yy, n, m);
  else
    hipLaunchKernelGGL((lora_join_kernel<kF16>), grid, block, 0, stream, l, part, splits, yy, n, m);
  return hipGetLastError();
}

}  // namespace imq
