// attention_tiles.hpp -- the matrix-core attention kernel and the kernel that
// joins its key ranges.
//
// A workgroup of NW waves holds NW * 32 rows of one sequence and key head,
// 32 a wave: row m is query m / G of head m % G of the G heads that share the
// key head, so keys and values are staged once for the whole group, and a few
// queries of many heads still fill a tile.  It walks the keys 64 at a time:
//
//   S^T [64 keys][32 rows] = K Q^T        2 * D/16 MFMAs of 32 x 32 x 16
//   P^T = exp2(S^T - max)                 32 values a lane, one row a lane pair
//   O^T [D][32 rows] += V^T P^T           4 * D/32 MFMAs
//
// The products are transposed so that a lane holds scores of one row only: the
// row's maximum and sum are a lane's own (joined with the lane 32 away), and
// the accumulator layout of S^T is, with the keys of a 16-key slice taken in
// the order 8 (e / 4) + 4 h + e % 4, the operand layout of P^T: the weights
// never leave their registers.  K and V tiles go straight from memory to LDS
// (16 bytes a lane, no registers), one tile ahead of the one in use; V's
// operand is read through the LDS transpose loads, 4 keys of 16 columns each.
// 16-byte pieces of a row are swizzled (XOR with the row) at their source, so
// the row-per-lane reads of K and the 4-row reads of V touch every bank evenly
// (no conflicts counted; the outputs' way through LDS has some).
//
// Two workgroups of four waves share a CU (64 KB of LDS and up to 256 registers a
// lane each), or one of eight has it, so that one wave of a SIMD multiplies while
// the other weighs: a tile of 64 keys is 32 MFMAs of 32 cycles a wave and some 130
// VALU instructions, 32 of them exponentials (8 cycles).  Measured, D = 128: 4608 x 4608 of 24 heads in f16 252-285 us
// (915-1035 TFLOP/s, the clock at 1.8 GHz; a large hipBLASLt product 1467), 16384 causal
// rows of 32 / 8 heads in bf16 1.97 ms (1114), with slopes 2.02-2.09.  The matrix cores
// are busy for half of the cycles.  With parts left out, the last took 2.05 ms of four
// waves a workgroup, 1.88 without the loads, 1.60 without the LDS reads, 1.65
// without the weighing: LDS, written and read, is what the rest waits for.
// Tried and slower: 256 rows in two groups of waves that take turns by
// barriers, the next scores' MFMAs among one wave's own exponentials, 64 rows of
// a workgroup where a CU gets more than one, V and K lines read ahead into L2.
#pragma once

#include "attention.hpp"

namespace imq {

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef short s16x8_t __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;

template <int T>
__device__ __forceinline__ f32x16_t attn_mfma(s16x8_t a, s16x8_t b, f32x16_t c) {
  if constexpr (T == kBf16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// A lane's value and that of the lane 32 away, in the same order in both.
// (The halves are taken as rvalues: bit-casting a vector's element in place
// reads element 0.)
__device__ __forceinline__ void lane_pair(float v, float& lo, float& hi) {
  const unsigned u = __builtin_bit_cast(unsigned, v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const unsigned a = r[0], b = r[1];
  lo = __builtin_bit_cast(float, a);
  hi = __builtin_bit_cast(float, b);
}
__device__ __forceinline__ float pair_max(float v) {
  float a, b;
  lane_pair(v, a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float pair_sum(float v) {
  float a, b;
  lane_pair(v, a, b);
  return a + b;
}

// Where in a row the 16-byte piece `piece` of row `row` lies in LDS.
template <int D>
__device__ __forceinline__ int k_piece(int row, int piece) {
  return D == 128 ? piece ^ (row & 15) : piece ^ ((row >> 1) & 7);
}
template <int D>
__device__ __forceinline__ int v_piece(int row, int piece) {
  return D == 128 ? piece ^ (4 * (row & 3)) : piece ^ (4 * ((row >> 1) & 1));
}

// What S^T accumulators of 32 keys start from.  A slope's fall is linear in the
// key before p: what it gives the keys of a tile apart from their first one is put
// there, divided by the factor that the scores take later, so that it costs nothing
// a score.  (A capped score is capped before it falls.)
template <bool kCap, bool kSlope>
__device__ __forceinline__ f32x16_t attn_start(const AttnScore<kCap, kSlope>& score) {
  f32x16_t c0;
#pragma unroll
  for (int e = 0; e < 16; ++e)
    c0[e] = kSlope && !kCap ? score.fall / score.mul * (float)(8 * (e / 4) + e % 4) : 0.f;
  return c0;
}

// The scores of 32 U keys (S^T accumulators, from attn_start) capped, lowered and
// masked; their row's largest, in units of log2.  j0: the first key; seen: the keys
// this lane's row sees; seen_lo: the fewest that any row of the wave sees; away0:
// p - j0 of the row.  What is left in sc is such that a key's exponent is
// sc * score.mul without a cap; with a cap alone, top - 2 top sc, as sc is the
// 1 / (exp(2 z) + 1) of the tanh (the exponent is one fma from it, made with the
// subtraction of the maximum); with cap and slope, sc; and with a slope, + shift[u],
// the part that 32 keys share.  Tiles that reach past p (none where causal hides
// those keys) take the distance itself.
template <int U, bool kCap, bool kSlope>
__device__ __forceinline__ float attn_scores(const AttnScore<kCap, kSlope>& score,
                                             f32x16_t (&sc)[U], int j0, int h, int seen,
                                             int seen_lo, int away0, bool linear,
                                             float (&shift)[U]) {
#pragma unroll
  for (int u = 0; u < U; ++u) shift[u] = 0.f;
  if constexpr (kSlope) {
    const float away = (float)(away0 - 4 * h);
    if (linear) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        shift[u] = -score.fall * (away - (float)(u * 32));
        if constexpr (kCap)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            sc[u][e] = __builtin_fmaf(score.fall, (float)(8 * (e / 4) + e % 4), score.capped(sc[u][e]));
      }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float key = (float)(8 * (e / 4) + e % 4), from = away - (float)(u * 32) - key;
          if constexpr (kCap) {
            sc[u][e] = score(sc[u][e], from);
          } else {
            const float x = __builtin_fmaf(-score.fall, key, sc[u][e] * score.mul);
            sc[u][e] = __builtin_fmaf(-score.fall, __builtin_fabsf(from), x) * (1.f / score.mul);
          }
        }
    }
  } else if constexpr (kCap) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[u][e] = score.rest(sc[u][e]);
  }
  constexpr bool kRest = kCap && !kSlope;  // falls with the score: a hidden key's is infinite
  if (j0 + 32 * U > seen_lo) {
    const int lim = seen - j0 - 4 * h;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        sc[u][e] = u * 32 + 8 * (e / 4) + e % 4 < lim ? sc[u][e] : kRest ? INFINITY : -INFINITY;
  }
  float mx;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float m = sc[u][0];
#pragma unroll
    for (int e = 1; e < 16; ++e) m = kRest ? fminf(m, sc[u][e]) : fmaxf(m, sc[u][e]);
    // mul is positive.
    if constexpr (kSlope) m = kCap ? m + shift[u] : __builtin_fmaf(m, score.mul, shift[u]);
    mx = u == 0 ? m : kRest ? fminf(mx, m) : fmaxf(mx, m);
  }
  if constexpr (kRest) mx = __builtin_fmaf(-2.f * score.top, mx, score.top);
  else if constexpr (!kSlope) mx *= score.mul;
  return pair_max(mx);
}

// How a weight is held until the sums are divided by the weights' own: exp2(score -
// top) times 2^kAttnLift, while top is behind the row's largest score by up to
// kAttnLag, so that the largest weight is between 2^kAttnLift and 2^(kAttnLift +
// kAttnLag).  f16 keeps 11 bits down to 2^-14 only and nothing under 2^-25: weights
// are lifted as far as it goes up (2^16), so that those down to 2^-25 of the row's
// largest keep their bits and none above 2^-36 is lost; at 2^0 to 2^8, 6000 keys 2^-25
// of the largest came to nothing.  bf16 has fp32's range: weights of 1 and less keep
// the products with its largest values in fp32, as far as the sums go.
template <int T>
constexpr float kAttnLag = T == kF16 ? 4.f : 8.f;
template <int T>
constexpr float kAttnLift = T == kF16 ? 11.f : -8.f;

// Moves the running maximum on, and the sums with it: only where a row's has
// grown by kAttnLag.
template <int T, int N>
__device__ __forceinline__ void attn_top(float mx, f32x16_t (&o)[N], float& top, float& sum) {
  if (__builtin_amdgcn_ballot_w64(mx > top + kAttnLag<T>)) {
    const float next = fmaxf(top, mx);
    const float keep = __builtin_amdgcn_exp2f(top - (next == -INFINITY ? 0.f : next));
    top = next;
    sum *= keep;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[i][e] *= keep;
  }
}

typedef float f32x2_t __attribute__((ext_vector_type(2)));

// Two weights to T.  In f16 as a vector: of two scalar conversions, among the
// sums of the same values, the compiler makes three instructions for one.
template <int T>
__device__ __forceinline__ uint32_t attn_pack2(float lo, float hi) {
  if constexpr (T == kF16)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{lo, hi}), f16x2_t));
  else
    return pack_bf16x2(lo, hi);
}

// x + the sum of the two T values of w, exactly added up in 32 bits.
template <int T>
__device__ __forceinline__ float attn_add2(uint32_t w, float x) {
  if constexpr (T == kF16) return dot2_f16(w, 0x3C003C00u, x);
  else return dot2_bf16(w, 0x3F803F80u, x);
}

// Scores to weights, exp2(score - top + kAttnLift): P^T fragments, and their sum.  The
// weights are rounded to T, what the matrix cores multiply: what that loses as a second
// product would be half as many products again, where they bind (the mean error against 64
// bits is 0.0019-0.0023 in bf16 and 0.00029 in f16, of weights kept in fp32 0.0016 and
// 0.00021).  The sum is that of the weights as rounded, which are what V is multiplied by;
// two a dot2 instruction.  kRest: a weight as two bf16, the second as fragments of
// its own, for a second product with V: its upper half, and what is left, with 2^-18 of
// all of them (which the division by the sum takes away) so that neither is zero where
// the weight is not: an infinite value stays what it is.
template <int T, int U, bool kCap, bool kSlope, bool kRest = false>
__device__ __forceinline__ void attn_weights(const AttnScore<kCap, kSlope>& score,
                                             const f32x16_t (&sc)[U], const float (&shift)[U],
                                             float top, float& sum, s16x8_t (&pf)[2 * U * (kRest ? 2 : 1)]) {
  // The exponent as one fma of what attn_scores left.
  const float by = !kCap ? score.mul : kSlope ? 1.f : -2.f * score.top;
  float add[2] = {sum, 0.f};
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const float base = (top == -INFINITY ? 0.f : top - kAttnLift<T>) -
                       (kSlope ? shift[u] : kCap ? score.top : 0.f);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t w[4], rest[4];
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float x0 = sc[u][half * 8 + e], x1 = sc[u][half * 8 + e + 1];
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(x0, by, -base));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(x1, by, -base));
        if constexpr (kRest) {
          const uint32_t b0 = __float_as_uint(p0) & 0xFFFF0000u, b1 = __float_as_uint(p1) & 0xFFFF0000u;
          w[e / 2] = b0 >> 16 | b1;
          rest[e / 2] = attn_pack2<T>(__builtin_fmaf(p0, 1.f + 0x1p-18f, -__uint_as_float(b0)),
                                      __builtin_fmaf(p1, 1.f + 0x1p-18f, -__uint_as_float(b1)));
          add[(e / 2) & 1] = attn_add2<T>(rest[e / 2], add[(e / 2) & 1]);
        } else {
          w[e / 2] = attn_pack2<T>(p0, p1);
        }
        add[(e / 2) & 1] = attn_add2<T>(w[e / 2], add[(e / 2) & 1]);
      }
      pf[u * 2 + half] = __builtin_bit_cast(s16x8_t, make_uint4(w[0], w[1], w[2], w[3]));
      if constexpr (kRest)
        pf[2 * U + u * 2 + half] = __builtin_bit_cast(s16x8_t, make_uint4(rest[0], rest[1], rest[2], rest[3]));
    }
  }
  sum = add[0] + add[1];
}

// S^T of 32 keys, added to c0: K rows from LDS (row c of the 32 at `lds`), Q^T from registers.
template <int T, int D>
__device__ __forceinline__ f32x16_t attn_qk(const uint4* lds, const s16x8_t (&qf)[D / 16], int c,
                                            int h, const f32x16_t& c0) {
  const int kf = D == 128 ? (c & 15) : ((c >> 1) & 7);  // k_piece's
  f32x16_t sc = c0;
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
    sc = attn_mfma<T>(__builtin_bit_cast(s16x8_t, lds[c * (D / 8) + ((2 * i + h) ^ kf)]), qf[i], sc);
  return sc;
}

// O^T += V^T P^T over 16 N keys: the rows at `lds` through the transpose loads
// (kRest: and the weights' remainders, N fragments behind the weights').
template <int T, int D, int N, bool kRest = false>
__device__ __forceinline__ void attn_pv(const uint4* lds, const s16x8_t (&pf)[N * (kRest ? 2 : 1)],
                                        f32x16_t (&o)[D / 32], int lane) {
  const int vr = 4 * (lane >> 5) + ((lane & 15) >> 2);           // of 8 rows
  const int vf = D == 128 ? 4 * (vr & 3) : 4 * ((vr >> 1) & 1);  // v_piece's
  const int vc = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);      // 16-byte piece of 32 columns
#pragma unroll
  for (int kc = 0; kc < N; ++kc)
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      s16x4_t part[2];
#pragma unroll
      for (int e4 = 0; e4 < 2; ++e4) {
        const int at = ((16 * kc + 8 * e4 + vr) * (D / 8) + ((4 * i + vc) ^ vf)) * 2 + (lane & 1);
        part[e4] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_s16x4_t*)(reinterpret_cast<const uint2*>(lds) + at));
      }
      const s16x8_t vv = __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
      o[i] = attn_mfma<T>(vv, pf[kc], o[i]);
      if constexpr (kRest) o[i] = attn_mfma<T>(vv, pf[N + kc], o[i]);
    }
}

// Q^T fragments of this lane's row: elements 16 i + 8 h to 16 i + 8 h + 8, zero past dim.
template <int T, int D>
__device__ __forceinline__ void attn_load_q(const AttnArgs& a, const AttnSeq& s, int t, int head,
                                            int h, s16x8_t (&qf)[D / 16]) {
  using S = typename Elem<T>::S;
  const S* q = static_cast<const S*>(a.q) + s.q_at + t * a.q_row + head * a.q_head;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    const int d = 16 * i + 8 * h;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (d < a.dim) v = *reinterpret_cast<const uint4*>(q + d);
    qf[i] = __builtin_bit_cast(s16x8_t, v);
  }
}

// A row's 64-bit offset from the lane that holds it.
__device__ __forceinline__ int64_t lane_offset(int64_t v, int from) {
  const uint32_t lo = __shfl((uint32_t)v, from, 64), hi = __shfl((uint32_t)(v >> 32), from, 64);
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// The wave's 32 rows between memory and a row a lane, through 32 rows of LDS of its
// own: memory sees whole rows, D / 8 lanes of 16 bytes each, where a row a lane
// touches 32 lines an instruction.  16 prompts of 512 rows, 32 / 8 heads, 69 us against
// 82 (with neither loads of Q nor stores, 43), 8 x 250 rows on 64 keys 13.4 / 14.9; not with
// 64 rows a workgroup, which are few and wait for LDS longer (4 x 120 on 64 keys
// 8.0 / 7.5), nor for Q with 256, whose LDS would not hold it, and with heads of 64
// elements, whose rows are a line each (level; the capped kernel would take 131
// registers, 99 us for 97).  Pieces are swizzled as k_piece's, by the row.
template <int D>
struct AttnRows {
  static constexpr int kLanes = D / 8, kRows = 64 / kLanes, kSteps = 32 / kRows;
  uint4* lds;
  int lane;
  __device__ __forceinline__ int row(int k) const { return k * kRows + lane / kLanes; }
  __device__ __forceinline__ int piece() const { return lane % kLanes; }
  __device__ __forceinline__ uint4& at(int row, int piece) const {
    return lds[row * kLanes + (piece ^ (row & (kLanes - 1)))];
  }
  // LDS of one wave is in order; this keeps the compiler to it.
  __device__ __forceinline__ void fence() const {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
};

template <int D>
struct AttnStage {
  uint4 k[kAttnKeys * D / 8];
  uint4 v[kAttnKeys * D / 8];
};

// One tile of `rows` (up to 64) rows of K or V into LDS: NW waves, D / (8 NW)
// loads each.  Pieces past the tensor's rows or the head's dim read as zero.
template <int D, int NW>
__device__ __forceinline__ void attn_load(const char* base, int64_t row_bytes, int rows, int dim,
                                          const uint32_t (&off)[D / (8 * NW)], uint4* lds, int wave) {
  // No rows: every read gives zero.
  const __amdgpu_buffer_rsrc_t rs =
      make_rsrc(base, rows > 0 ? (uint32_t)((rows - 1) * row_bytes + dim * 2) : 0u);
#pragma unroll
  for (int i = 0; i < D / (8 * NW); ++i) load_lds16(rs, off[i], 0, lds + (i * NW + wave) * 64);
}

// Waves of a workgroup with WM of them on rows of their own.
constexpr int attn_waves(int wm) { return wm < 4 ? 4 : wm; }

template <int T, int D, int WM, bool kCap, bool kSlope, bool kSplit>
__global__ __launch_bounds__(attn_waves(WM) * 64, 2) void attn_tiles_kernel(
    AttnArgs a, int tiles, int first, int near_hs, int splits, int chunk, float* ws) {
  using S = typename Elem<T>::S;
  // WM waves on rows of their own, WK on a part of every tile's keys each.
  constexpr int NW = attn_waves(WM), WK = NW / WM, U = 2 / WK, kRows = WM * 32;
  constexpr int kLoads = D / (8 * NW);
  __shared__ AttnStage<D> st0, st1;
  __shared__ float qs[NW][D];
  const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hs_n = a.n_seq * a.kv_heads;
  // near_hs sequences and key heads (all, where keys are split) at a time.
  const int hs0 = kSplit ? 0 : blockIdx.x / (near_hs * tiles) * near_hs;
  const int hs_now = kSplit ? hs_n : min(near_hs, hs_n - hs0);
  const int at = blockIdx.x - hs0 * tiles;
  const int hs = hs0 + at % hs_now, rest = at / hs_now;
  const int split = kSplit ? rest % splits : 0;
  // The last rows of a causal sequence have the most keys: they start first.
  // Where every workgroup is resident from the start, two a CU, those behind
  // the first `first` ranks, which get a CU's second place, go from the least
  // keys up instead, so that a long one shares its CU with a short one.
  const int rank = kSplit ? rest / splits : rest;
  const int tile = rank < first ? tiles - 1 - rank : rank - first;
  const int kh = hs % a.kv_heads;
  AttnSeq s = attn_seq(a, hs / a.kv_heads);
  const int group = a.heads / a.kv_heads;
  const int rows = s.nq * group;  // checked on the host to fit
  const int m0 = tile * kRows;
  if (m0 >= rows) return;
  // Rows past the last repeat it; they are not stored.
  const int wm = wave % WM, wk = wave / WM;
  const int mw = m0 + wm * 32;
  const int m = min(mw + c, rows - 1);
  const int t = m / group, head = kh * group + m % group;
  const int seen = attn_seen(a, s, t);
  const int seen_wg = __builtin_amdgcn_readfirstlane(
      attn_seen(a, s, min(m0 + kRows - 1, rows - 1) / group));
  const int seen_hi = mw >= rows ? 0 : __builtin_amdgcn_readfirstlane(
      attn_seen(a, s, min(mw + 31, rows - 1) / group));
  const int seen_lo = __builtin_amdgcn_readfirstlane(attn_seen(a, s, min(mw, rows - 1) / group));
  const int begin = kSplit ? split * chunk : 0;
  const int end = kSplit ? min(seen_wg, begin + chunk) : seen_wg;
  if (kSplit && begin >= end) return;  // the join reads the ranges up to seen_wg only

  // Sources of this thread's pieces in a tile.
  const int64_t kb = a.k_row * 2, vb = a.v_row * 2;
  uint32_t k_off[kLoads], v_off[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int at = (i * NW + wave) * 64 + lane, row = at / (D / 8), piece = at % (D / 8);
    const int kp = k_piece<D>(row, piece), vp = v_piece<D>(row, piece);
    k_off[i] = kp * 8 < a.dim ? (uint32_t)(row * kb + kp * 16) : 0x80000000u;
    v_off[i] = vp * 8 < a.dim ? (uint32_t)(row * vb + vp * 16) : 0x80000000u;
  }
  const char* kbase = reinterpret_cast<const char*>(static_cast<const S*>(a.k) + s.k_at + kh * a.k_head);
  const char* vbase = reinterpret_cast<const char*>(static_cast<const S*>(a.v) + s.v_at + kh * a.v_head);
  auto issue = [&](AttnStage<D>& st, int j0) {
    // Nothing past the last tile: rows below 1.
    const int n = j0 < end ? min(kAttnKeys, s.nk - j0) : 0;
    attn_load<D, NW>(kbase + j0 * kb, kb, n, a.dim, k_off, st.k, wave);
    attn_load<D, NW>(vbase + j0 * vb, vb, n, a.dim, v_off, st.v, wave);
  };
  s16x8_t qf[D / 16];
  if constexpr (WM == 4 && D == 128) {
    // st1 is free until the first tile is in use.
    const AttnRows<D> part{reinterpret_cast<uint4*>(&st1) + wave * (32 * D / 8), lane};
    const S* q = static_cast<const S*>(a.q) + s.q_at;
    const int64_t q_off = t * a.q_row + head * a.q_head;
    uint4 v[AttnRows<D>::kSteps];
#pragma unroll
    for (int k = 0; k < AttnRows<D>::kSteps; ++k) {
      const int64_t off = lane_offset(q_off, part.row(k));
      v[k] = make_uint4(0, 0, 0, 0);
      if (part.piece() * 8 < a.dim) v[k] = *reinterpret_cast<const uint4*>(q + off + part.piece() * 8);
    }
    if (begin < end) issue(st0, begin);
#pragma unroll
    for (int k = 0; k < AttnRows<D>::kSteps; ++k) part.at(part.row(k), part.piece()) = v[k];
    part.fence();
#pragma unroll
    for (int i = 0; i < D / 16; ++i) qf[i] = __builtin_bit_cast(s16x8_t, part.at(c, 2 * i + h));
  } else {
    if (begin < end) issue(st0, begin);
    attn_load_q<T, D>(a, s, t, head, h, qf);
  }
  const AttnScore<kCap, kSlope> score(a, head);
  const f32x16_t c0 = attn_start(score);
  const int p = t + s.nk - s.nq;
  // Keys below `near` are at or before every row's p, or hidden behind it.
  const int near = a.causal && !a.prefix_lens ? INT_MAX : min(mw, rows - 1) / group + s.nk - s.nq + 1;
  f32x16_t o[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
  float top = -INFINITY, sum = 0.f;

  // The wave's keys of the tile that begins at j0.
  // The next tile's loads go out among the score's MFMAs: before them they
  // would hold up the wave that has everyone wait.
  auto step = [&](const AttnStage<D>& st, AttnStage<D>& to, int j0) __attribute__((always_inline)) {
    const int j1 = j0 + kAttnKeys;
    j0 += wk * (32 * U);
    if (j0 >= seen_hi) {
      issue(to, j1);
      return;
    }
    const uint4* k = st.k + wk * U * 32 * (D / 8);
    f32x16_t sc[U];
#pragma unroll
    for (int u = 0; u < U; ++u) sc[u] = attn_qk<T, D>(k + u * 32 * (D / 8), qf, c, h, c0);
    issue(to, j1);
    // K of eight MFMAs is read ahead: one read an MFMA, as the compiler has
    // it, leaves most of an LDS read's 100 to 200 cycles exposed.
    constexpr int kReads = U * D / 16, kAhead = kReads < 8 ? kReads : 8;
    __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
    for (int i = 0; i < kReads - kAhead; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x20, 1, 0);
    }
    s16x8_t pf[2 * U];
    float shift[U];
    attn_top<T>(attn_scores<U, kCap, kSlope>(score, sc, j0, h, seen, seen_lo, p - j0,
                                             j0 + 32 * U <= near, shift), o, top, sum);
    attn_weights<T, U, kCap, kSlope>(score, sc, shift, top, sum, pf);
    attn_pv<T, D, 2 * U>(st.v + wk * U * 32 * (D / 8), pf, o, lane);
  };

  // A tile in use, the next in flight.  Every wave's loads of a stage have
  // landed, and its reads of the other are done, once all have met.
  auto meet = [&] {
    __builtin_amdgcn_sched_barrier(0);
    IMQ_WAIT_VM_LGKM_0();
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  for (int j0 = begin; j0 < end; j0 += 2 * kAttnKeys) {
    meet();
    step(st0, st1, j0);
    if (j0 + kAttnKeys >= end) break;
    meet();
    step(st1, st0, j0 + kAttnKeys);
  }
  IMQ_WAIT_VMCNT(0);  // the loads past the last tile (of nothing), before their LDS is used again
  __builtin_amdgcn_sched_barrier(0);

  sum = pair_sum(sum);
  if constexpr (WK == 2) {
    // The second half's sums through the stages' LDS, lane for lane.
    static_assert(sizeof(AttnStage<D>) >= WM * 64 * (D / 2) * 4, "a wave's sums fit half a stage");
    float4* po = reinterpret_cast<float4*>(&st0) + wm * (D / 8) * 64 + lane;
    float2* pt = reinterpret_cast<float2*>(&st1) + wm * 64 + lane;
    meet();
    if (wk == 1) {
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          po[(i * 4 + e / 4) * 64] = make_float4(o[i][e], o[i][e + 1], o[i][e + 2], o[i][e + 3]);
      *pt = make_float2(top, sum);
    }
    meet();
    if (wk == 1) return;
    const float2 other = *pt;
    const float next = fmaxf(top, other.x);
    const float base = next == -INFINITY ? 0.f : next;
    const float keep0 = __builtin_amdgcn_exp2f(top - base), keep1 = __builtin_amdgcn_exp2f(other.x - base);
    top = next;
    sum = sum * keep0 + other.y * keep1;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const float4 v = po[(i * 4 + e / 4) * 64];
        o[i][e] = o[i][e] * keep0 + v.x * keep1;
        o[i][e + 1] = o[i][e + 1] * keep0 + v.y * keep1;
        o[i][e + 2] = o[i][e + 2] * keep0 + v.z * keep1;
        o[i][e + 3] = o[i][e + 3] * keep0 + v.w * keep1;
      }
  }
  if constexpr (kSplit) {
    // [split][row of all tiles][D], then (top, sum) of each.
    const int64_t all = (int64_t)hs_n * tiles * kRows;
    const int64_t row = ((int64_t)hs * tiles + tile) * kRows + wm * 32 + c;
    if (mw + c < rows) {
      float* po = ws + ((int64_t)split * all + row) * D;
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          *reinterpret_cast<float4*>(po + i * 32 + 2 * e + 4 * h) =
              make_float4(o[i][e], o[i][e + 1], o[i][e + 2], o[i][e + 3]);
      if (h == 0)
        *reinterpret_cast<float2*>(ws + (int64_t)splits * all * D +
                                   ((int64_t)split * all + row) * 2) = make_float2(top, sum);
    }
  } else {
    // (Of keys whose scores are all -infinity the sum is zero too, and the output NaN.)
    const float inv = seen > 0 ? 1.f / sum : 0.f;
    bool finite = true;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        o[i][e] *= inv;
        finite = finite && __builtin_fabsf(o[i][e]) < INFINITY;
      }
    S* out = static_cast<S*>(a.out) + s.out_at;
    const int64_t out_off = t * a.out_row + head * a.out_head;
    auto packed = [&](int i, int e) {
      return make_uint2(Elem<T>::pack2(o[i][e], o[i][e + 1]), Elem<T>::pack2(o[i][e + 2], o[i][e + 3]));
    };
    if constexpr (WK == 1) {
      meet();  // through the LDS where the tiles were
      const AttnRows<D> part{reinterpret_cast<uint4*>(wm < 4 ? &st0 : &st1) + wm % 4 * (32 * D / 8), lane};
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          reinterpret_cast<uint2*>(&part.at(c, i * 4 + e / 4))[h] = packed(i, e);
      part.fence();
#pragma unroll
      for (int k = 0; k < AttnRows<D>::kSteps; ++k) {
        const int64_t off = lane_offset(out_off, part.row(k));
        const uint4 v = part.at(part.row(k), part.piece());
        if (mw + part.row(k) < rows && part.piece() * 8 < a.dim)
          *reinterpret_cast<uint4*>(out + off + part.piece() * 8) = v;
      }
    } else if (mw + c < rows) {
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const int d = i * 32 + 2 * e + 4 * h;
          if (d < a.dim) *reinterpret_cast<uint2*>(out + out_off + d) = packed(i, e);
        }
    }
    uint64_t again = __builtin_amdgcn_ballot_w64(!finite && sum == sum && mw + c < rows);
    if (again) {
      const int odd = attn_spoilt<T>(a, s, kh, seen_lo, seen_hi + kAttnKeys);
      again = __builtin_amdgcn_ballot_w64(!finite && sum == sum && mw + c < rows && seen <= odd);
    }
    again = (again | again >> 32) & 0xFFFFFFFFu;
    while (again) {
      const int r = __builtin_ctzll(again);
      again &= again - 1;
      const int tr = (mw + r) / group;
      attn_row<T, kCap, kSlope>(a, s, kh * group + (mw + r) % group, tr, attn_seen(a, s, tr), qs[wave]);
    }
  }
}

// Joins the key ranges of a split plan: 16 lanes a row, D / 16 columns each,
// kParts such groups a row that take the ranges in turn (range i is group
// i % kParts's) and are joined through LDS in order.  tile_rows rows a tile; a
// tile's ranges up to the last key that its last row sees are written, the
// others not.  Bound by the latency of its loads: four ranges a group are in
// flight together.
template <int T, int D, int kParts, bool kCap, bool kSlope>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a, int tile_rows, int tiles,
                                                        int splits, int chunk, const float* ws) {
  using S = typename Elem<T>::S;
  __shared__ float qs[4][D];
  __shared__ float sums[kParts > 1 ? 16 : 1][D + 2];
  // Read with the first arguments, not each where it is used.
  asm volatile("" ::"s"(ws), "s"(splits), "s"(chunk), "s"(tile_rows), "s"(a.out), "s"(a.causal),
               "s"(a.max_q), "s"(a.max_k), "s"(a.out_row), "s"(a.out_head), "s"(a.prefix_lens));
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, slot = threadIdx.x / 16;
  const int64_t all = (int64_t)a.n_seq * a.kv_heads * tiles * tile_rows;
  const int64_t row = (int64_t)blockIdx.x * (16 / kParts) + slot / kParts;
  const int part = slot % kParts;
  const int group = a.heads / a.kv_heads;
  const int64_t of_seq = (int64_t)tiles * tile_rows;
  bool live = row < all;
  const int hs = (int)((live ? row : 0) / of_seq);
  const int m = (int)((live ? row : 0) % of_seq);
  const AttnSeq s = attn_seq(a, hs / a.kv_heads);
  const int kh = hs % a.kv_heads;
  const int rows = s.nq * group;
  live = live && m < rows;
  const int t = m / group, head = kh * group + m % group;
  const int d0 = (lane & 15) * (D / 16);
  float acc[D / 16] = {}, top = -INFINITY, sum = 0.f;
  if (live) {
    const int last = min(m / tile_rows * tile_rows + tile_rows, rows) - 1;
    const int used = (int)(((int64_t)attn_seen(a, s, last / group) + chunk - 1) / chunk);
    const float2* ml = reinterpret_cast<const float2*>(ws + (int64_t)splits * all * D) + row;
    const float* po = ws + row * D + d0;
    for (int i = part; i < used; i += 4 * kParts) {
      float2 v[4];
      float4 w[4][D / 64];
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int64_t at = (int64_t)min(i + b * kParts, used - 1) * all;
        v[b] = ml[at];
#pragma unroll
        for (int e = 0; e < D / 64; ++e) w[b][e] = reinterpret_cast<const float4*>(po + at * D)[e];
      }
      float next = top;
#pragma unroll
      for (int b = 0; b < 4; ++b) next = fmaxf(next, v[b].x);
      const float base = next == -INFINITY ? 0.f : next;
      const float old = __builtin_amdgcn_exp2f(top - base);
      top = next;
      sum *= old;
#pragma unroll
      for (int e = 0; e < D / 16; ++e) acc[e] *= old;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        if (i + b * kParts >= used) break;
        const float keep = __builtin_amdgcn_exp2f(v[b].x - base);
        sum = __builtin_fmaf(v[b].y, keep, sum);
#pragma unroll
        for (int e = 0; e < D / 64; ++e) {
          acc[4 * e] = __builtin_fmaf(w[b][e].x, keep, acc[4 * e]);
          acc[4 * e + 1] = __builtin_fmaf(w[b][e].y, keep, acc[4 * e + 1]);
          acc[4 * e + 2] = __builtin_fmaf(w[b][e].z, keep, acc[4 * e + 2]);
          acc[4 * e + 3] = __builtin_fmaf(w[b][e].w, keep, acc[4 * e + 3]);
        }
      }
    }
  }
  if constexpr (kParts > 1) {
#pragma unroll
    for (int e = 0; e < D / 16; ++e) sums[slot][d0 + e] = acc[e];
    if ((lane & 15) == 0) {
      sums[slot][D] = top;
      sums[slot][D + 1] = sum;
    }
    __syncthreads();
    const int s0 = slot - part;
    live = live && part == 0;
    if (live) {
#pragma unroll
      for (int b = 1; b < kParts; ++b) top = fmaxf(top, sums[s0 + b][D]);
      const float base = top == -INFINITY ? 0.f : top;
      sum = 0.f;
#pragma unroll
      for (int e = 0; e < D / 16; ++e) acc[e] = 0.f;
#pragma unroll
      for (int b = 0; b < kParts; ++b) {
        const float keep = __builtin_amdgcn_exp2f(sums[s0 + b][D] - base);
        sum = __builtin_fmaf(sums[s0 + b][D + 1], keep, sum);
#pragma unroll
        for (int e = 0; e < D / 16; ++e) acc[e] = __builtin_fmaf(sums[s0 + b][d0 + e], keep, acc[e]);
      }
    }
  }
  bool again_row = false;
  if (live) {
    const float inv = attn_seen(a, s, t) > 0 ? 1.f / sum : 0.f;
    S* out = static_cast<S*>(a.out) + s.out_at + t * a.out_row + head * a.out_head;
#pragma unroll
    for (int e = 0; e < D / 16; ++e) {
      acc[e] *= inv;
      again_row = again_row || !(__builtin_fabsf(acc[e]) < INFINITY);
    }
    again_row = again_row && sum == sum;
#pragma unroll
    for (int e = 0; e < D / 16; e += 4)
      if (d0 + e < a.dim)
        *reinterpret_cast<uint2*>(out + d0 + e) =
            make_uint2(Elem<T>::pack2(acc[e], acc[e + 1]), Elem<T>::pack2(acc[e + 2], acc[e + 3]));
  }
  uint64_t again = __builtin_amdgcn_ballot_w64(again_row);
  if (again == 0) return;
  const AttnArgs a1 = attn_args_again();
  while (again) {
    const int l = __builtin_ctzll(again) & ~15;
    again &= ~(0xFFFFull << l);
    const int mr = __builtin_amdgcn_readlane(m, l), hr = __builtin_amdgcn_readlane(hs, l);
    const AttnSeq sr = attn_seq(a1, hr / a1.kv_heads);
    const int tr = mr / group, seen = attn_seen(a1, sr, tr), khr = hr % a1.kv_heads;
    const int last = min(mr / tile_rows * tile_rows + tile_rows, sr.nq * group) - 1;
    if (seen <= attn_spoilt<T>(a1, sr, khr, seen, attn_seen(a1, sr, last / group) + kAttnKeys))
      attn_row<T, kCap, kSlope>(a1, sr, khr * group + mr % group, tr, seen, qs[wave]);
  }
}

}  // namespace imq
