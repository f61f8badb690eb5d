// attention_walk.hpp -- the tiles of attention_tiles.hpp and their join behind shared keys.  Kernels
// of their own: with these steps among its own the plain ones took up to a tenth longer (16 x 512
// rows of 32 / 8 heads 67.8 us for 61.8), other registers and another order of the same loop.
#pragma once

#include <type_traits>

#include "attention.hpp"
#include "attention_tiles.hpp"

namespace imq {

// Where the own keys begin in a walk over shared and own ones: behind whole pairs of tiles.
__device__ __forceinline__ int attn_own0(const AttnShared& sh) {
  return (sh.rows + 2 * kAttnKeys - 1) / (2 * kAttnKeys) * (2 * kAttnKeys);
}

// Sums of ranges of shared keys.
struct AttnFront {
  const float* ws;  // as a split plan's, of `all` rows
  int64_t all;
  int ranges;
  int packed;  // rows of a key head, which stand in q's order; 0: the same rows as other ranges
};
__device__ __forceinline__ int64_t attn_packed_row(const AttnArgs& a, const AttnFront& front, int seq, int kh,
                                                   int t, int g) {
  const int64_t q = (a.q_offsets ? (int64_t)min(max(a.q_offsets[seq], 0), a.q_rows) : (int64_t)seq * a.max_q) + t;
  return (int64_t)kh * front.packed + q * (a.heads / a.kv_heads) + g;
}

// What stands before every sequence's keys: the keys of an AttnShared, which the walk begins with,
// or their sums, which it goes on from.
struct AttnSums {
  AttnShared sh;
  AttnFront front;
};
// attn_tiles_kernel's tiles behind shared keys; what is said of those holds here too.
template <int T, int D, int WM, bool kCap, bool kSlope, bool kSplit, class Before>
__global__ __launch_bounds__(attn_waves(WM) * 64, 2) void attn_walk_kernel(
    AttnArgs a, int tiles, int first, int near_hs, int splits, int chunk, float* ws, Before before) {
  constexpr bool kShared = std::is_same_v<Before, AttnShared>, kSums = std::is_same_v<Before, AttnSums>;
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
  int own0 = 0;
  if constexpr (kShared) own0 = attn_own0(before);
  const int begin = kSplit ? split * chunk : 0;
  const int end = kSplit ? min(own0 + seen_wg, begin + chunk) : own0 + seen_wg;
  if (kSplit && begin >= end) return;  // the join reads the ranges up to seen_wg only

  // Sources of this thread's pieces in a tile.
  const int64_t kb = a.k_row * 2, vb = a.v_row * 2;
  uint32_t k_off[kLoads], v_off[kLoads];
  auto sources = [&](int64_t kb, int64_t vb) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int at = (i * NW + wave) * 64 + lane, row = at / (D / 8), piece = at % (D / 8);
      const int kp = k_piece<D>(row, piece), vp = v_piece<D>(row, piece);
      k_off[i] = kp * 8 < a.dim ? (uint32_t)(row * kb + kp * 16) : 0x80000000u;
      v_off[i] = vp * 8 < a.dim ? (uint32_t)(row * vb + vp * 16) : 0x80000000u;
    }
  };
  sources(kb, vb);
  const char* kbase = reinterpret_cast<const char*>(static_cast<const S*>(a.k) + s.k_at + kh * a.k_head);
  const char* vbase = reinterpret_cast<const char*>(static_cast<const S*>(a.v) + s.v_at + kh * a.v_head);
  // Among the shared keys: their sources, until the own ones' turn.
  const char *now_k = kbase - own0 * kb, *now_v = vbase - own0 * vb;  // of the walk's key 0
  int64_t now_kb = kb, now_vb = vb;
  int now_end = own0 + s.nk;
  int front_rows = 0;
  if constexpr (kShared) {
    front_rows = before.rows;
    if (begin < own0) {
      now_k = static_cast<const char*>(before.k) + kh * before.k_head * 2, now_kb = before.k_row * 2;
      now_v = static_cast<const char*>(before.v) + kh * before.v_head * 2, now_vb = before.v_row * 2;
      now_end = before.rows;
      sources(now_kb, now_vb);
    }
  }
  auto issue = [&](AttnStage<D>& st, int j0) {
    // Nothing past the last tile: rows below 1.
    if constexpr (kShared) {
      const int n = j0 < end ? min(kAttnKeys, now_end - j0) : 0;
      attn_load<D, NW>(now_k + j0 * now_kb, now_kb, n, a.dim, k_off, st.k, wave);
      attn_load<D, NW>(now_v + j0 * now_vb, now_vb, n, a.dim, v_off, st.v, wave);
    } else {
      const int n = j0 < end ? min(kAttnKeys, s.nk - j0) : 0;
      attn_load<D, NW>(kbase + j0 * kb, kb, n, a.dim, k_off, st.k, wave);
      attn_load<D, NW>(vbase + j0 * vb, vb, n, a.dim, v_off, st.v, wave);
    }
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
  if constexpr (kSums) {
    static_assert(WK == 1, "every wave has its rows alone");
    const AttnFront& front = before.front;
    const int64_t at = attn_packed_row(a, front, hs / a.kv_heads, kh, t, m % group);
    const float2* ml = reinterpret_cast<const float2*>(front.ws + front.ranges * front.all * D) + at;
    for (int r = 0; r < front.ranges; ++r) {
      const float2 v = ml[r * front.all];
      const float* po = front.ws + (r * front.all + at) * D;
      const float next = fmaxf(top, v.x), base = next == -INFINITY ? 0.f : next;
      const float keep0 = __builtin_amdgcn_exp2f(top - base), keep1 = __builtin_amdgcn_exp2f(v.x - base);
      top = next;
      sum = sum * keep0 + (h == 0 ? v.y * keep1 : 0.f);  // the lane 32 away's is added at the end
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const float4 w = *reinterpret_cast<const float4*>(po + i * 32 + 2 * e + 4 * h);
          o[i][e] = o[i][e] * keep0 + w.x * keep1;
          o[i][e + 1] = o[i][e + 1] * keep0 + w.y * keep1;
          o[i][e + 2] = o[i][e + 2] * keep0 + w.z * keep1;
          o[i][e + 3] = o[i][e + 3] * keep0 + w.w * keep1;
        }
    }
  }

  // The wave's keys of the tile that begins at j0.
  // The next tile's loads go out among the score's MFMAs: before them they
  // would hold up the wave that has everyone wait.
  auto step = [&](auto in_front, const AttnStage<D>& st, AttnStage<D>& to,
                  int j0) __attribute__((always_inline)) {
    constexpr bool front = decltype(in_front)::value;
    const int j1 = j0 + kAttnKeys;
    // What the rows see of the walk, where they stand in it, and `near`, among the shared
    // keys and among the own ones.
    if (front && j1 == own0) {
      now_k = kbase - own0 * kb, now_kb = kb;
      now_v = vbase - own0 * vb, now_vb = vb;
      now_end = own0 + s.nk;
      sources(kb, vb);
    }
    const int walk_seen = front ? front_rows : own0 + seen, walk_lo = front ? front_rows : own0 + seen_lo;
    const int walk_hi = front ? (mw >= rows ? 0 : front_rows) : own0 + seen_hi;
    const int walk_p = p + (front ? front_rows : own0);
    const int walk_near = front ? min(mw, rows - 1) / group + s.nk - s.nq + 1 + front_rows
                          : near == INT_MAX ? near : own0 + near;
    j0 += wk * (32 * U);
    if (j0 >= walk_hi) {
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
    // Weights rounded to T once, as attention's tiles have them: mean error 0.0023 in bf16 for 0.0014 with
    // what is left as a second fragment (the streams' form), but 74 us for 92 of 16 x 128 rows behind 2048 keys,
    // 919 for 1155 of 4 x 2048 behind 8192: the matrix cores have no time to spare here.
    s16x8_t pf[2 * U];
    float shift[U];
    attn_top<T>(attn_scores<U, kCap, kSlope>(score, sc, j0, h, walk_seen, walk_lo, walk_p - j0,
                                             j0 + 32 * U <= walk_near, shift), o, top, sum);
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
  // (Two loops: with one, whose steps tell the keys apart, 4 x 2048 rows of 32 / 8 heads behind
  // 8192 shared keys took 1293 us for 1275.)
  auto go = [&](auto in_front, int from, int to) __attribute__((always_inline)) {
    for (int j0 = from; j0 < to; j0 += 2 * kAttnKeys) {
      meet();
      step(in_front, st0, st1, j0);
      if (j0 + kAttnKeys >= to) break;
      meet();
      step(in_front, st1, st0, j0 + kAttnKeys);
    }
  };
  if constexpr (kShared) {
    go(std::true_type{}, begin, min(own0, end));
    go(std::false_type{}, max(begin, own0), end);
  } else {
    go(std::false_type{}, begin, end);
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
    const float inv = 1.f / sum;
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
      const AttnRows<D> part{reinterpret_cast<uint4*>(&st0) + wm * (32 * D / 8), lane};
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
      const AttnShared* sh;
      if constexpr (kSums) sh = &before.sh;
      else sh = &before;
      attn_row_shared<T, kCap, kSlope>(a, *sh, s, kh * group + (mw + r) % group, tr, attn_seen(a, s, tr), qs[wave]);
    }
  }
}

// attn_join_kernel's join behind shared keys: a row's first front.ranges ranges are the shared
// keys', and the others are counted from `own0` keys before its own.
struct AttnJoinShared {
  AttnShared sh;
  AttnFront front;
  int own0;
};
template <int T, int D, int kParts, bool kCap, bool kSlope>
__global__ __launch_bounds__(256) void attn_shared_join_kernel(AttnArgs a, int tile_rows, int tiles, int splits,
                                                               int chunk, const float* ws, AttnJoinShared before) {
  const AttnFront& front = before.front;
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
    const int used = front.ranges +
                     (int)(((int64_t)attn_seen(a, s, last / group) + before.own0 + chunk - 1) / chunk);
    const float2* ml = reinterpret_cast<const float2*>(ws + (int64_t)splits * all * D) + row;
    const float* po = ws + row * D + d0;
    const float2* front_ml =
        reinterpret_cast<const float2*>(front.ws + (int64_t)front.ranges * front.all * D) + row;
    const float* front_po = front.ws + row * D + d0;
    for (int i = part; i < used; i += 4 * kParts) {
      float2 v[4];
      float4 w[4][D / 64];
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int range = min(i + b * kParts, used - 1);
        const bool in_front = range < front.ranges;
        const int64_t at = in_front ? range * front.all : (range - front.ranges) * all;
        v[b] = (in_front ? front_ml : ml)[at];
#pragma unroll
        for (int e = 0; e < D / 64; ++e)
          w[b][e] = reinterpret_cast<const float4*>((in_front ? front_po : po) + at * D)[e];
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
    const float inv = 1.f / sum;
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
      attn_row_shared<T, kCap, kSlope>(a1, before.sh, sr, khr * group + mr % group, tr, seen, qs[wave]);
  }
}

}  // namespace imq
