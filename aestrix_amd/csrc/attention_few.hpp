// attention_few.hpp -- attention of up to 32 rows (queries times the heads of a
// key head) over a long range of keys: single tokens over a cache.
//
// Bound by reading K and V once.  The products are those of
// attention_tiles.hpp on one 32-row tile, whose matrix work is an eighth of
// what the memory takes; so nothing is shared: each of a workgroup's four
// waves walks key tiles of its own, 32 keys (tiles 4 n + wave of the range),
// with its own LDS and no barrier.  K and V have one buffer each and take turns:
// K of the next tile is loaded while the softmax and the product with V run, V
// while the next scores are made, so 8 to 16 KB a wave are in flight, four
// waves a CU (one workgroup, where keys are split).  The four waves' sums are joined through LDS at the end.
// 131072 keys of 8 key heads: 93 us, 5.8 TB/s (and 5.2 for the join; the tiles'
// kernel 149 in all); 8 sequences of up to 2048 keys: 9.1 us, from the MALL, and 4.0.
#pragma once

#include <type_traits>

#include "attention_tiles.hpp"

namespace imq {

template <int T, int D, bool kCap, bool kSlope, bool kSplit>
__global__ __launch_bounds__(kFewWaves * 64, 2) void attn_few_kernel(AttnArgs a, int tile_rows,
                                                                    int splits, int chunk, float* ws) {
  using S = typename Elem<T>::S;
  constexpr int kPieces = kFewKeys * D / 8, kLoads = kPieces / 64;
  // bf16 weights carry 8 bits, and a second bf16 of each what that leaves, up to 2^-7
  // of it, multiplied with V as well: the matrix cores have the time.  (f16
  // weights lose 2^-12, or 2^-36 of the row's largest where that is more.)
  constexpr bool kRest = T == kBf16;
  __shared__ uint4 kbuf[kFewWaves][kPieces];
  __shared__ uint4 vbuf[kFewWaves][kPieces];
  __shared__ float2 ml[kFewWaves][32];
  __shared__ unsigned bad;
  const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hs_n = a.n_seq * a.kv_heads;
  const int hs = blockIdx.x % hs_n;
  const int split = kSplit ? blockIdx.x / hs_n : 0;
  const int kh = hs % a.kv_heads;
  const AttnSeq s = attn_seq(a, hs / a.kv_heads);
  const int group = a.heads / a.kv_heads;
  const int rows = s.nq * group;
  if (rows == 0) return;
  const int m = min(c, rows - 1);
  const int t = m / group, head = kh * group + m % group;
  const int seen = attn_seen(a, s, t);
  const int seen_hi = __builtin_amdgcn_readfirstlane(attn_seen(a, s, s.nq - 1));
  const int seen_lo = __builtin_amdgcn_readfirstlane(attn_seen(a, s, 0));
  const int begin = kSplit ? split * chunk : 0;
  const int end = kSplit ? min(seen_hi, begin + chunk) : seen_hi;
  if (kSplit && begin >= end) return;  // the join reads the ranges up to seen_hi only

  const int64_t kb = a.k_row * 2, vb = a.v_row * 2;
  uint32_t k_off[kLoads], v_off[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int at = i * 64 + lane, row = at / (D / 8), piece = at % (D / 8);
    const int kp = k_piece<D>(row, piece), vp = v_piece<D>(row, piece);
    k_off[i] = kp * 8 < a.dim ? (uint32_t)(row * kb + kp * 16) : 0x80000000u;
    v_off[i] = vp * 8 < a.dim ? (uint32_t)(row * vb + vp * 16) : 0x80000000u;
  }
  const char* kbase = reinterpret_cast<const char*>(static_cast<const S*>(a.k) + s.k_at + kh * a.k_head);
  const char* vbase = reinterpret_cast<const char*>(static_cast<const S*>(a.v) + s.v_at + kh * a.v_head);
  auto load = [&](const char* base, int64_t row_bytes, const uint32_t (&off)[kLoads], uint4* lds, int j0) {
    const int n = min(kFewKeys, s.nk - j0);  // 0 where there are no keys: all reads give zero
    const __amdgpu_buffer_rsrc_t rs = make_rsrc(
        base + j0 * row_bytes, n > 0 ? (uint32_t)((n - 1) * row_bytes + a.dim * 2) : 0u);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load_lds16(rs, off[i], 0, lds + i * 64);
  };
  uint4* kl = kbuf[wave];
  uint4* vl = vbuf[wave];
  constexpr int kStep = kFewWaves * kFewKeys;
  const int first = begin + wave * kFewKeys;
  s16x8_t qf[D / 16];
  attn_load_q<T, D>(a, s, t, head, h, qf);
  __builtin_amdgcn_sched_barrier(0);
  // Also in a wave without a tile (the range's last one then): the counts of
  // loads in flight below hold on every path.
  load(kbase, kb, k_off, kl, max(min(first, end - 1), 0));
  load(vbase, vb, v_off, vl, max(min(first, end - 1), 0));
  __builtin_amdgcn_sched_barrier(0);
  const AttnScore<kCap, kSlope> score(a, head);
  const f32x16_t c0 = attn_start(score);
  const int p = t + s.nk - s.nq;
  // Keys below `near` are at or before every row's p, or hidden behind it.
  const int near = a.causal && !a.prefix_lens ? INT_MAX : s.nk - s.nq + 1;
  f32x16_t o[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
  float top = -INFINITY, sum = 0.f;
  __builtin_amdgcn_sched_barrier(0);
  IMQ_WAIT_VMCNT(2 * kLoads);  // q is in registers
  __builtin_amdgcn_sched_barrier(0);
  // One tile; kMore: and the next one's loads.  (Not a condition inside the
  // loop: with a path that skips only some loads the compiler waits for all.)
  auto step = [&](auto more, int j0) {
    constexpr bool kMore = decltype(more)::value;
    // K has landed when only this tile's V is in flight.
    __builtin_amdgcn_sched_barrier(0);
    IMQ_WAIT_VMCNT(kLoads);
    __builtin_amdgcn_sched_barrier(0);
    f32x16_t sc[1];
    sc[0] = attn_qk<T, D>(kl, qf, c, h, c0);
    __builtin_amdgcn_sched_barrier(0);
    IMQ_WAIT_LGKM_0();  // K has been read
    if constexpr (kMore) load(kbase, kb, k_off, kl, j0 + kStep);
    __builtin_amdgcn_sched_barrier(0);
    s16x8_t pf[kRest ? 4 : 2];
    float shift[1];
    attn_top<T>(attn_scores<1, kCap, kSlope>(score, sc, j0, h, seen, seen_lo, p - j0,
                                             j0 + kFewKeys <= near, shift), o, top, sum);
    attn_weights<T, 1, kCap, kSlope, kRest>(score, sc, shift, top, sum, pf);
    __builtin_amdgcn_sched_barrier(0);
    IMQ_WAIT_VMCNT(kMore ? kLoads : 0);  // V has landed (the next K is in flight)
    __builtin_amdgcn_sched_barrier(0);
    attn_pv<T, D, 2, kRest>(vl, pf, o, lane);
    __builtin_amdgcn_sched_barrier(0);
    IMQ_WAIT_LGKM_0();  // V has been read
    if constexpr (kMore) load(vbase, vb, v_off, vl, j0 + kStep);
    __builtin_amdgcn_sched_barrier(0);
  };
  int j0 = first;
  for (; j0 + kStep < end; j0 += kStep) step(std::true_type{}, j0);
  if (j0 < end) step(std::false_type{}, j0);

  IMQ_WAIT_VMCNT(0);  // an idle wave's loads too, before their buffers are used again
  __builtin_amdgcn_sched_barrier(0);
  // Rows 0-15 of a wave's sums into its K buffer, 16-31 into its V buffer.
  sum = pair_sum(sum);
  float* part = reinterpret_cast<float*>(c < 16 ? kbuf[wave] : vbuf[wave]) + (c & 15) * D;
  if (c < rows) {
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *reinterpret_cast<float4*>(part + i * 32 + 2 * e + 4 * h) =
            make_float4(o[i][e], o[i][e + 1], o[i][e + 2], o[i][e + 3]);
    if (h == 0) ml[wave][c] = make_float2(top, sum);
  }
  if (threadIdx.x == 0) bad = 0;
  __syncthreads();
  constexpr int kPer = D / 4;  // threads of a row, four columns each
  const int64_t all = (int64_t)hs_n * tile_rows;
  for (int r = threadIdx.x / kPer; r < rows; r += kFewWaves * 64 / kPer) {
    const int d = threadIdx.x % kPer * 4;
    float tops = -INFINITY;
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) tops = fmaxf(tops, ml[w][r].x);
    const float base = tops == -INFINITY ? 0.f : tops;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sums = 0.f;
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) {
      const float keep = __builtin_amdgcn_exp2f(ml[w][r].x - base);
      sums = __builtin_fmaf(ml[w][r].y, keep, sums);
      const float4 v = *reinterpret_cast<const float4*>(
          reinterpret_cast<const float*>(r < 16 ? kbuf[w] : vbuf[w]) + (r & 15) * D + d);
      acc.x = __builtin_fmaf(v.x, keep, acc.x);
      acc.y = __builtin_fmaf(v.y, keep, acc.y);
      acc.z = __builtin_fmaf(v.z, keep, acc.z);
      acc.w = __builtin_fmaf(v.w, keep, acc.w);
    }
    if constexpr (kSplit) {
      const int64_t at = (int64_t)split * all + (int64_t)hs * tile_rows + r;
      *reinterpret_cast<float4*>(ws + at * D + d) = acc;
      if (d == 0)
        *reinterpret_cast<float2*>(ws + (int64_t)splits * all * D + at * 2) = make_float2(tops, sums);
    } else {
      const float inv = attn_seen(a, s, r / group) > 0 ? 1.f / sums : 0.f;
      acc.x *= inv, acc.y *= inv, acc.z *= inv, acc.w *= inv;
      const float big = fmaxf(fmaxf(__builtin_fabsf(acc.x), __builtin_fabsf(acc.y)),
                              fmaxf(__builtin_fabsf(acc.z), __builtin_fabsf(acc.w)));
      const bool nan = acc.x != acc.x || acc.y != acc.y || acc.z != acc.z || acc.w != acc.w;
      if ((nan || big == INFINITY) && sums == sums) atomicOr(&bad, 1u << r);
      S* out = static_cast<S*>(a.out) + s.out_at + (r / group) * a.out_row +
               (kh * group + r % group) * a.out_head;
      if (d < a.dim)
        *reinterpret_cast<uint2*>(out + d) = make_uint2(Elem<T>::pack2(acc.x, acc.y),
                                                        Elem<T>::pack2(acc.z, acc.w));
    }
  }
  if constexpr (!kSplit) {
    __syncthreads();
    float* qs = reinterpret_cast<float*>(kbuf[wave]);
    const int odd = bad ? attn_spoilt<T>(a, s, kh, seen_lo, seen_hi + kFewKeys) : -1;
    for (unsigned again = bad; again; again &= again - 1) {
      const int r = __builtin_ctz(again);
      const int tr = r / group, of = attn_seen(a, s, tr);
      if (r % kFewWaves != wave || of > odd) continue;
      attn_row<T, kCap, kSlope>(a, s, kh * group + r % group, tr, of, qs);
    }
  }
}

}  // namespace imq
