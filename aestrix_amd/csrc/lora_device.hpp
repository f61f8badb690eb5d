// lora_device.hpp -- device code of adapters beside the quantized matmul
// (include/imq_lora.h) and the tile kernels' output stage with them.
#pragma once

#include <climits>
#include <type_traits>

#include "epilogue.hpp"
#include "imq_device.hpp"
#include "lora.hpp"

namespace imq {

// Adapter i's first row of A, and its rank (whatever `first` holds, inside A and B).
struct LoraAt {
  int row, rank;
};
__device__ __forceinline__ LoraAt lora_at(const LoraArgs& l, int i) {
  const int a = min(max(l.first[i], 0), l.rows) & ~15, b = min(max(l.first[i + 1], a), l.rows);
  return LoraAt{a, min(b - a, l.max_rank) & ~15};
}
// The adapter of row `row` (< m), or -1.
__device__ __forceinline__ int lora_of(const LoraArgs& l, int row) {
  const int i = l.which[row];
  return (unsigned)i < (unsigned)l.count ? i : -1;
}

// What A's row `row`, one of adapter i's, is multiplied by.
__device__ __forceinline__ float lora_scale(const LoraArgs& l, int i, int row) {
  return l.scale[l.rank_scales ? row : i];
}

// u of row `row` and rank `rank` to its place: the upper half, and what it leaves (nothing where
// it is infinite).
template <int T>
__device__ __forceinline__ void lora_put(const LoraArgs& l, int row, int rank, float u) {
  const uint16_t hi = Elem<T>::out(u);
  const float v = staged_value<T>(hi);
  const uint16_t lo = Elem<T>::out(__builtin_fabsf(v) < INFINITY ? u - v : 0.f);
  uint16_t* to = l.u + (((size_t)(row / 32) * (l.max_rank / 16) + rank / 16) * 2 * 64 + row % 32 +
                        32 * (rank >> 3 & 1)) * 8 + (rank & 7);
  to[0] = hi;
  to[64 * 8] = lo;
}

// u of row at / max_rank and rank at % max_rank (of few rows), by a wave.  Bound by reading A, and
// by the latency of that: kAhead pieces of 1 KB of each of the two rows are on their way together (64
// rows of K = 9728, rank 16, 24 adapters: 7.2 us).
template <int T, int kAhead>
__device__ __forceinline__ void lora_dot(const LoraArgs& l, const uint16_t* x, int k, int m, int at) {
  const int lane = threadIdx.x & 63;
  const int row = at / l.max_rank, r = at % l.max_rank;
  if (row >= m) return;
  const int i = lora_of(l, row);
  if (i < 0) return;
  const LoraAt to = lora_at(l, i);
  if (r >= to.rank) return;
  const __amdgpu_buffer_rsrc_t ar = make_rsrc(l.a + (size_t)(to.row + r) * k, (uint32_t)k * 2);
  const int from = l.order ? l.order[row] : row;
  const __amdgpu_buffer_rsrc_t xr = make_rsrc(x + (size_t)from * k, (uint32_t)k * 2);
  float sum[2] = {0.f, 0.f};
  for (int c = 0; c < k; c += kAhead * 512) {
    u32x4_t av[kAhead], xv[kAhead];  // (past the end: zeros)
#pragma unroll
    for (int p = 0; p < kAhead; ++p) {
      av[p] = load_b128(ar, lane * 16, (uint32_t)c * 2 + p * 1024);
      xv[p] = load_b128(xr, lane * 16, (uint32_t)c * 2 + p * 1024);
    }
    __builtin_amdgcn_sched_barrier(0);  // all of them first, rather than few for more waves
#pragma unroll
    for (int p = 0; p < kAhead; ++p)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        sum[e & 1] = T == kBf16 ? dot2_bf16(av[p][e], xv[p][e], sum[e & 1])
                                : dot2_f16(av[p][e], xv[p][e], sum[e & 1]);
  }
  float u = sum[0] + sum[1];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) u += __shfl_xor(u, off, 64);
  if (lane == 0) lora_put<T>(l, row, r, u * lora_scale(l, i, to.row + r));
}

// u's first fragment of 32 rows (tile) for this lane: the first 16 ranks' upper halves.
__device__ __forceinline__ const u32x4_t* lora_u(const LoraArgs& l, int tile) {
  return reinterpret_cast<const u32x4_t*>(l.u) + (size_t)tile * (l.max_rank / 16) * 128 + (threadIdx.x & 63);
}

template <int T>
__device__ __forceinline__ f32x16_t lora_mfma(u32x4_t a, u32x4_t b, f32x16_t c) {
  if constexpr (T == kBf16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// c = B_i u of 32 rows (tile) and 32 columns from n0 on, in the accumulators' layout.
// B's rows come straight from memory in operand layout: a lane's column and eight ranks are 16
// bytes.
template <int T>
__device__ __forceinline__ f32x16_t lora_product(const LoraArgs& l, const LoraAt& at, int tile, int n0, int N) {
  const int lane = threadIdx.x & 63, r32 = lane & 31, h = lane >> 5;
  const u32x4_t* b = reinterpret_cast<const u32x4_t*>(l.b + (size_t)at.row * N +
                                                      (size_t)min(n0 + r32, N - 1) * at.rank) + h;
  f32x16_t c;
#pragma unroll
  for (int e = 0; e < 16; ++e) c[e] = 0.f;
  const u32x4_t* u = lora_u(l, tile);
  for (int r = 0; r < at.rank / 16; ++r) {
    const u32x4_t hi = u[r * 128], lo = u[r * 128 + 64], bv = b[2 * r];
    c = lora_mfma<T>(hi, bv, c);
    c = lora_mfma<T>(lo, bv, c);
  }
  return c;
}

// The smallest of the wave's values.
__device__ __forceinline__ int lora_least(int v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = min(v, __shfl_xor(v, off, 64));
  return __builtin_amdgcn_readfirstlane(v);
}

// Two values of T, those that are not finite as zero; odd: raised where there are any.
template <int T>
__device__ __forceinline__ uint32_t lora_finite(uint32_t v, uint32_t& odd) {
  constexpr uint32_t kExp = T == kBf16 ? 0x7F80u : 0x7C00u;
  const uint32_t bad = ((v & kExp) == kExp ? 0xFFFFu : 0u) | ((v >> 16 & kExp) == kExp ? 0xFFFF0000u : 0u);
  odd |= bad;
  return v & ~bad;
}

// acc[mt][nt] += B u of the rows from m0 (a multiple of 32) and the columns from n0 on, 32 x 32
// each, in the accumulators' layout.  lds: MT * 8 KB that the whole workgroup of four waves is
// done with once it meets; every wave has the same rows.
//
// u of the workgroup's rows comes to LDS, 64 ranks at a time, straight from memory.  Then the
// adapters that the rows name one after the other, the product of all rows with each: for every
// 16 ranks B's fragments, straight from memory in operand layout (a lane's column and eight ranks
// are 16 bytes) and one product ahead.  A row that names another adapter has u = 0 here, and of B
// what is not finite is zero too, so that an adapter's NaN stays with its rows; they are NaN in
// that column.  (A product apart from the accumulators, added row by row, had the compiler move
// 192 of 256 accumulators about in every iteration of the K loop, 478 us for 418.)
template <int T, int MT, int NT>
__device__ __forceinline__ void lora_tail(const LoraArgs& l, f32x16_t (&acc)[MT][NT], uint4* lds, int m0,
                                          int n0, int M, int N) {
  constexpr int kWaves = 4, kBlock = 4;  // 16-rank chunks at a time
  const int lane = threadIdx.x & 63, r32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int id[MT], least = INT_MAX;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int row = m0 + mt * 32 + r32;
    id[mt] = row < M ? lora_of(l, row) : -1;
    least = min(least, id[mt] < 0 ? INT_MAX : id[mt]);
  }
  const int i0 = lora_least(least);
  if (i0 == INT_MAX) return;
  auto after = [&](int i) {
    int v = INT_MAX;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) v = min(v, id[mt] > i ? id[mt] : INT_MAX);
    return lora_least(v);
  };
  // u from this tile on; past the end zeros.
  const uint32_t per = (uint32_t)l.max_rank / 16 * 2048;  // bytes of 32 rows
  const __amdgpu_buffer_rsrc_t ur =
      make_rsrc(reinterpret_cast<const char*>(l.u) + (size_t)(m0 / 32) * per,
                (uint32_t)min(MT, (M + 31) / 32 - m0 / 32) * per);
  for (int r0 = 0; r0 < l.max_rank / 16; r0 += kBlock) {
    // Every wave is done with this LDS, and nothing of its own is on its way there.
    __builtin_amdgcn_sched_barrier(0);
    IMQ_WAIT_VM_LGKM_0();
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int p = 0; p < kBlock * MT * 2 / kWaves; ++p) {
      const int at = p * kWaves + wave, c = at / (2 * MT), mt = at / 2 % MT, part = at % 2;
      load_lds16(ur, lane * 16, mt * per + (r0 + c) * 2048 + part * 1024, lds + at * 64);
    }
    u32x4_t bf[NT];
    auto load_b = [&](const LoraAt& at, int r) {
      if (at.rank == 0) return;
      r = min(r, at.rank / 16 - 1);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        bf[nt] = *reinterpret_cast<const u32x4_t*>(l.b + (size_t)at.row * N +
                                                   (size_t)min(n0 + nt * 32 + r32, N - 1) * at.rank +
                                                   16 * r + 8 * h);
    };
    LoraAt at = lora_at(l, i0);
    load_b(at, r0);
    __builtin_amdgcn_sched_barrier(0);
    IMQ_WAIT_VMCNT(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    for (int i = i0;;) {
      const int next = after(i);
      const LoraAt then = next == INT_MAX ? at : lora_at(l, next);
      const int chunks = min(at.rank / 16 - r0, kBlock);
      if (chunks <= 0) load_b(then, r0);
      uint32_t odd[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) odd[nt] = 0;
      for (int c = 0; c < chunks; ++c) {
        u32x4_t bn[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) bn[nt][e] = lora_finite<T>(bf[nt][e], odd[nt]);
        if (c + 1 < chunks) load_b(at, r0 + c + 1);
        else load_b(then, r0);
#pragma unroll
        for (int part = 0; part < 2; ++part)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            const u32x4_t u = __builtin_bit_cast(u32x4_t, lds[((c * MT + mt) * 2 + part) * 64 + lane]);
            const u32x4_t a = id[mt] == i ? u : u32x4_t{0u, 0u, 0u, 0u};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) acc[mt][nt] = lora_mfma<T>(a, bn[nt], acc[mt][nt]);
          }
      }
      uint32_t any = 0;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) any |= odd[nt];
      if (__builtin_amdgcn_ballot_w64(any != 0)) {
        // NaN where a row that names it meets such a column, by matrix instructions alone:
        // bf16's largest value squared, which is infinite, less the same.
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const uint64_t cols = __builtin_amdgcn_ballot_w64(odd[nt] != 0);  // a column's ranks are in two lanes
          const uint32_t col = (uint32_t)(cols | cols >> 32) >> r32 & 1u ? 0x7F7F7F7Fu : 0u;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int sign = 0; sign < 2; ++sign) {
              const uint32_t row = id[mt] == i ? (sign ? 0xFF7FFF7Fu : 0x7F7F7F7Fu) : 0u;
              acc[mt][nt] = lora_mfma<kBf16>(u32x4_t{row, row, row, row}, u32x4_t{col, col, col, col}, acc[mt][nt]);
            }
        }
      }
      if (next == INT_MAX) break;
      i = next, at = then;
    }
  }
}

// EpStore with the adapters' products added to the sums.
template <int T>
struct EpLora : EpStore<T> {
  LoraArgs lora;
  __device__ __forceinline__ int row_at(int place) const { return lora.order ? lora.order[place] : place; }
  __device__ __forceinline__ void emit1(int row, int col, uint16_t v) const {
    EpStore<T>::emit1(row_at(row), col, v);
  }
  __device__ __forceinline__ void emit8(int row, int col, uint4 v) const {
    EpStore<T>::emit8(row_at(row), col, v);
  }
  template <int MT, int NT>
  __device__ __forceinline__ void add_sums(f32x16_t (&acc)[MT][NT], uint4* lds, int m0, int n0, int M,
                                           int N) const {
    lora_tail<T, MT, NT>(lora, acc, lds, m0, n0, M, N);
  }
};
template <int T>
constexpr bool adds_sums<EpLora<T>> = true;

}  // namespace imq
