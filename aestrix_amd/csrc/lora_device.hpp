// lora_device.hpp -- device code of adapters beside the quantized matmul
// (include/imq_lora.h) and the tile kernels' output stage with them.
#pragma once

#include "epilogue.hpp"
#include "imq_device.hpp"
#include "lora.hpp"

namespace imq {

// Adapter i's first row of A, and its rank (whatever `first` holds, inside A and B).
struct LoraAt {
  int row, rank;
};
__device__ __forceinline__ LoraAt lora_at(const LoraArgs& l, int i) {
  const int a = min(max(l.first[i], 0), l.rows), b = min(max(l.first[i + 1], a), l.rows);
  return LoraAt{a, min(b - a, l.max_rank) & ~15};
}
// The adapter of row `row` (< m), or -1.
__device__ __forceinline__ int lora_of(const LoraArgs& l, int row) {
  const int i = l.which[row];
  return (unsigned)i < (unsigned)l.count ? i : -1;
}

// Eight values of u as two of T each: the upper halves, and what they leave.
template <int T>
__device__ __forceinline__ void lora_split(const float* u, u32x4_t& hi, u32x4_t& lo) {
  const float4 a = reinterpret_cast<const float4*>(u)[0], b = reinterpret_cast<const float4*>(u)[1];
  const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    hi[e] = Elem<T>::pack2(v[2 * e], v[2 * e + 1]);
    const float h0 = staged_value<T>(hi[e] & 0xFFFFu), h1 = staged_value<T>(hi[e] >> 16);
    // (Infinite as T: nothing is left, rather than a NaN.)
    lo[e] = Elem<T>::pack2(__builtin_fabsf(h0) < INFINITY ? v[2 * e] - h0 : 0.f,
                           __builtin_fabsf(h1) < INFINITY ? v[2 * e + 1] - h1 : 0.f);
  }
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

// acc[mt][nt] += B u of the rows from m0 and the columns from n0 on (32 x 32 each, in
// the accumulators' layout).  Of every 32 rows the adapters that they name one after the
// other: the product of all 32 rows' u with B_i, B's rows straight from memory in operand
// layout (a lane's column and eight ranks are 16 bytes), and then that of the rows that
// name it added: a product of its own, so that an adapter's NaN stays with its rows.
template <int T, int MT, int NT>
__device__ __forceinline__ void lora_tail(const LoraArgs& l, f32x16_t (&acc)[MT][NT], int m0, int n0,
                                          int M, int N) {
  const int lane = threadIdx.x & 63, r32 = lane & 31, h = lane >> 5;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int row = m0 + mt * 32 + r32;
    const int id = row < M ? lora_of(l, row) : -1;
    const float* u = l.u + (size_t)min(row, M - 1) * l.max_rank + 8 * h;
    uint32_t left = (uint32_t)__builtin_amdgcn_ballot_w64(id >= 0);
    while (left) {
      const int i = __builtin_amdgcn_readlane(id, __builtin_ctz(left));
      const uint32_t rows = (uint32_t)__builtin_amdgcn_ballot_w64(id == i);
      left &= ~rows;
      const LoraAt at = lora_at(l, i);
      const uint16_t* b[NT];
      f32x16_t c[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        b[nt] = l.b + (size_t)at.row * N + (size_t)min(n0 + nt * 32 + r32, N - 1) * at.rank + 8 * h;
#pragma unroll
        for (int e = 0; e < 16; ++e) c[nt][e] = 0.f;
      }
      for (int r = 0; r < at.rank; r += 16) {
        u32x4_t hi, lo;
        lora_split<T>(u + r, hi, lo);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const u32x4_t bv = *reinterpret_cast<const u32x4_t*>(b[nt] + r);
          c[nt] = lora_mfma<T>(hi, bv, c[nt]);
          c[nt] = lora_mfma<T>(lo, bv, c[nt]);
        }
      }
      const uint32_t mine = rows >> (4 * h);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          acc[mt][nt][e] += (mine >> (8 * (e >> 2) + (e & 3))) & 1u ? c[nt][e] : 0.f;
    }
  }
}

// EpStore with the adapters' products added to the sums.
template <int T>
struct EpLora : EpStore<T> {
  LoraArgs lora;
  template <int MT, int NT>
  __device__ __forceinline__ void add_sums(f32x16_t (&acc)[MT][NT], int m0, int n0, int M, int N) const {
    lora_tail<T, MT, NT>(lora, acc, m0, n0, M, N);
  }
};
template <int T>
constexpr bool adds_sums<EpLora<T>> = true;

}  // namespace imq
