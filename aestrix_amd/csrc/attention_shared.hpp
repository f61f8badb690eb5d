// attention_shared.hpp -- softmax attention of sequences that begin with the same keys
// (imq_attention_shared, include/imq_core.h): kernels and launches, instantiated per
// element type in attention_shared_{bf16,f16}.hip.
//
// Sequences with many rows (queries times the heads of a key head) run the tiles of
// attention_walk.hpp, whose walk goes over the shared keys and then the own ones: the
// matrix cores bind there, and the shared keys come out of the caches (4 x up to 2048 rows of
// 32 / 8 heads of 128 behind 8192 keys, with slopes, 848-872 us, 940-966 TFLOP/s; of 6.0 GB of requests
// 0.18 pass the L2s).  Sequences that
// fill little of their tiles: all rows in one stretch against the shared keys first (launch_packed; 61
// documents of up to 154 rows, capped, behind 3001 keys 76 us, 119 in tiles of their own; 64 x 36 rows
// behind 8192 124 and 213).
//
// Up to 32 rows a sequence, single tokens mostly, are bound by reading keys.  So that the
// shared ones are read once for the batch, the rows of all sequences stand together
// against them, 32 or 64 a workgroup, and each sequence's own rows against its own keys, as
// workgroups of one launch (attn_stream_kernel); a second one joins the ranges.  Tokens of 32 / 8 heads
// of 128: 16 behind 65536 keys 60 us and the join 6, 286 MB past the L2s, 4.7 TB/s; 64 behind
// 8192, with up to 1024 own ones, 54 and 5, 173 MB, 3.2 TB/s (the shared ones are read four times, three
// of them out of the L2s: 280 MB of requests); 8 behind 512 7.5 and 4.5, the latency of a tile or two and of
// the join's loads.
#pragma once

#include <type_traits>

#include "attention.hpp"
#include "attention_tiles.hpp"
#include "attention_walk.hpp"
#include "imq_core.h"

namespace imq {

// ---- few rows a sequence

// With R = 2 the queries lie in LDS, as the fragments that a wave reads, and two workgroups
// have all of a CU's: what the end needs takes their place.
template <int D, int R>
struct StreamLds {
  uint4 k[kFewWaves][kFewKeys * D / 8];
  uint4 v[kFewWaves][kFewKeys * D / 8];
  union {
    uint4 q[R > 1 ? R * D / 16 : 1][64];
    struct {
      float2 ml[kFewWaves][32];
      int dst[32];
    } end;
  };
};

// Keys at k and v, `rows` of them that may be read.
struct StreamKeys {
  const char *k, *v;
  int64_t kb, vb;  // bytes from row to row
  int rows;
};

// 32 R rows against the keys [begin, end), begin < end: their sums, not yet divided, to
// row dst of po (D floats) and pml (top, sum); below 0: nowhere.  The products are those of
// attention_tiles.hpp.  Nothing is shared on the way: each of the four waves walks key tiles
// of its own, 32 keys (tiles 4 n + wave), with its own LDS and no barrier.  K and V have one
// buffer each and take turns: K of the next tile is loaded while the weights and the product
// with V are made, V while the next scores are.  With R = 2 a fragment of K or V is read from
// LDS once for two MFMAs.
template <int T, int D, int R, int kLdsR, bool kCap, bool kSlope>
__device__ __forceinline__ void attn_stream(const AttnArgs& a, StreamLds<D, kLdsR>& lds, const StreamKeys& keys,
                                            int begin, int end, const s16x8_t (&qf)[R][D / 16],
                                            const AttnScore<kCap, kSlope> (&score)[R], const int (&seen)[R],
                                            int seen_lo, const int (&p)[R], int near,
                                            const int (&dst)[R], float* po, float2* pml) {
  constexpr int kPieces = kFewKeys * D / 8, kLoads = kPieces / 64;
  // bf16 weights as two bf16 each, as in attn_few_kernel: the matrix cores have the time.
  constexpr bool kRest = T == kBf16;
  constexpr int kFrags = kRest ? 4 : 2;
  const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t k_off[kLoads], v_off[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int at = i * 64 + lane, row = at / (D / 8), piece = at % (D / 8);
    const int kp = k_piece<D>(row, piece), vp = v_piece<D>(row, piece);
    k_off[i] = kp * 8 < a.dim ? (uint32_t)(row * keys.kb + kp * 16) : 0x80000000u;
    v_off[i] = vp * 8 < a.dim ? (uint32_t)(row * keys.vb + vp * 16) : 0x80000000u;
  }
  auto load = [&](const char* base, int64_t row_bytes, const uint32_t (&off)[kLoads], uint4* to, int j0) {
    const int n = min(kFewKeys, keys.rows - j0);  // 0 where there are no keys: all reads give zero
    const __amdgpu_buffer_rsrc_t rs = make_rsrc(
        base + j0 * row_bytes, n > 0 ? (uint32_t)((n - 1) * row_bytes + a.dim * 2) : 0u);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load_lds16(rs, off[i], 0, to + i * 64);
  };
  uint4* kl = lds.k[wave];
  uint4* vl = lds.v[wave];
  constexpr int kStep = kFewWaves * kFewKeys;
  const int first = begin + wave * kFewKeys;
  __builtin_amdgcn_sched_barrier(0);
  // Also in a wave without a tile (the range's last one then): the counts of loads in
  // flight below hold on every path.
  load(keys.k, keys.kb, k_off, kl, min(first, end - 1));
  load(keys.v, keys.vb, v_off, vl, min(first, end - 1));
  __builtin_amdgcn_sched_barrier(0);
  f32x16_t o[R][D / 32];
  float top[R], sum[R];
#pragma unroll
  for (int g = 0; g < R; ++g) {
    top[g] = -INFINITY, sum[g] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[g][i][e] = 0.f;
  }
  __builtin_amdgcn_sched_barrier(0);
  IMQ_WAIT_VMCNT(2 * kLoads);  // what the caller loaded is in registers
  __builtin_amdgcn_sched_barrier(0);
  if constexpr (R > 1) {
#pragma unroll
    for (int g = 0; g < R; ++g)
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
        if (i % kFewWaves == wave) lds.q[g * (D / 16) + i][lane] = __builtin_bit_cast(uint4, qf[g][i]);
    __builtin_amdgcn_sched_barrier(0);
    IMQ_WAIT_LGKM_0();
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
  }
  const int kf = D == 128 ? (c & 15) : ((c >> 1) & 7);           // k_piece's
  const int vr = 4 * (lane >> 5) + ((lane & 15) >> 2);           // of 8 rows
  const int vf = D == 128 ? 4 * (vr & 3) : 4 * ((vr >> 1) & 1);  // v_piece's
  const int vc = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);      // 16-byte piece of 32 columns
  // One tile; kMore: and the next one's loads.
  auto step = [&](auto more, int j0) __attribute__((always_inline)) {
    constexpr bool kMore = decltype(more)::value;
    __builtin_amdgcn_sched_barrier(0);
    IMQ_WAIT_VMCNT(kLoads);  // K has landed (this tile's V is in flight)
    __builtin_amdgcn_sched_barrier(0);
    f32x16_t sc[R][1];
#pragma unroll
    for (int g = 0; g < R; ++g) {
      // Made anew for every tile: kept, it takes 16 registers a row that there are not.
      AttnScore<kCap, kSlope> from = score[g];
      if constexpr (kSlope && !kCap) asm volatile("" : "+v"(from.fall));
      sc[g][0] = attn_start(from);
    }
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      const s16x8_t kv = __builtin_bit_cast(s16x8_t, kl[c * (D / 8) + ((2 * i + h) ^ kf)]);
#pragma unroll
      for (int g = 0; g < R; ++g) {
        const s16x8_t qv = R > 1 ? __builtin_bit_cast(s16x8_t, lds.q[g * (D / 16) + i][lane]) : qf[g][i];
        sc[g][0] = attn_mfma<T>(kv, qv, sc[g][0]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    IMQ_WAIT_LGKM_0();  // K has been read
    if constexpr (kMore) load(keys.k, keys.kb, k_off, kl, j0 + kStep);
    __builtin_amdgcn_sched_barrier(0);
    s16x8_t pf[R][kFrags];
#pragma unroll
    for (int g = 0; g < R; ++g) {
      float shift[1];
      attn_top<T>(attn_scores<1, kCap, kSlope>(score[g], sc[g], j0, h, seen[g], seen_lo, p[g] - j0,
                                               j0 + kFewKeys <= near, shift), o[g], top[g], sum[g]);
      attn_weights<T, 1, kCap, kSlope, kRest>(score[g], sc[g], shift, top[g], sum[g], pf[g]);
    }
    __builtin_amdgcn_sched_barrier(0);
    IMQ_WAIT_VMCNT(kMore ? kLoads : 0);  // V has landed (the next K is in flight)
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int kc = 0; kc < 2; ++kc)
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        s16x4_t part[2];
#pragma unroll
        for (int e4 = 0; e4 < 2; ++e4) {
          const int at = ((16 * kc + 8 * e4 + vr) * (D / 8) + ((4 * i + vc) ^ vf)) * 2 + (lane & 1);
          part[e4] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lds_s16x4_t*)(reinterpret_cast<const uint2*>(vl) + at));
        }
        const s16x8_t vv = __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
        for (int g = 0; g < R; ++g) {
          o[g][i] = attn_mfma<T>(vv, pf[g][kc], o[g][i]);
          if constexpr (kRest) o[g][i] = attn_mfma<T>(vv, pf[g][2 + kc], o[g][i]);
        }
      }
    __builtin_amdgcn_sched_barrier(0);
    IMQ_WAIT_LGKM_0();  // V has been read
    if constexpr (kMore) load(keys.v, keys.vb, v_off, vl, j0 + kStep);
    __builtin_amdgcn_sched_barrier(0);
  };
  int j0 = first;
  for (; j0 + kStep < end; j0 += kStep) step(std::true_type{}, j0);
  if (j0 < end) step(std::false_type{}, j0);
  IMQ_WAIT_VMCNT(0);  // an idle wave's loads too, before their buffers are used again
  __builtin_amdgcn_sched_barrier(0);

  // The waves' sums joined, 32 rows at a time: rows 0-15 of a wave's into its K buffer, 16-31
  // into its V buffer.
#pragma unroll
  for (int g = 0; g < R; ++g) {
    if (R > 1) __syncthreads();  // the queries, or the last 32 rows, have been read
    const float total = pair_sum(sum[g]);
    float* part = reinterpret_cast<float*>(c < 16 ? lds.k[wave] : lds.v[wave]) + (c & 15) * D;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *reinterpret_cast<float4*>(part + i * 32 + 2 * e + 4 * h) =
            make_float4(o[g][i][e], o[g][i][e + 1], o[g][i][e + 2], o[g][i][e + 3]);
    if (h == 0) lds.end.ml[wave][c] = make_float2(top[g], total);
    if (threadIdx.x < 32) lds.end.dst[c] = dst[g];
    __syncthreads();
    constexpr int kPer = D / 4;  // threads of a row, four columns each
#pragma unroll
    for (int r = threadIdx.x / kPer; r < 32; r += kFewWaves * 64 / kPer) {
      const int64_t to = lds.end.dst[r];
      if (to < 0) continue;
      const int d = threadIdx.x % kPer * 4;
      float tops = -INFINITY;
#pragma unroll
      for (int w = 0; w < kFewWaves; ++w) tops = fmaxf(tops, lds.end.ml[w][r].x);
      const float base = tops == -INFINITY ? 0.f : tops;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      float sums = 0.f;
#pragma unroll
      for (int w = 0; w < kFewWaves; ++w) {
        const float keep = __builtin_amdgcn_exp2f(lds.end.ml[w][r].x - base);
        sums = __builtin_fmaf(lds.end.ml[w][r].y, keep, sums);
        const float4 v = *reinterpret_cast<const float4*>(
            reinterpret_cast<const float*>(r < 16 ? lds.k[w] : lds.v[w]) + (r & 15) * D + d);
        acc.x = __builtin_fmaf(v.x, keep, acc.x);
        acc.y = __builtin_fmaf(v.y, keep, acc.y);
        acc.z = __builtin_fmaf(v.z, keep, acc.z);
        acc.w = __builtin_fmaf(v.w, keep, acc.w);
      }
      *reinterpret_cast<float4*>(po + to * D + d) = acc;
      if (d == 0) pml[to] = make_float2(tops, sums);
    }
  }
}

// Every sequence's rows (rows: queries times heads a key head, up to 32) against the shared
// keys, then against their own: first kv_heads * s_tiles * s_splits workgroups of 32 R rows of
// the batch and s_chunk shared keys, then one for a sequence, key head and o_chunk own keys.
// The ranges of the shared keys go to ws, those of the own ones behind them, each as a split
// plan's.
template <int T, int D, int R, bool kCap, bool kSlope>
__global__ __launch_bounds__(kFewWaves * 64, 2) void attn_stream_kernel(
    AttnArgs a, AttnShared sh, int rows, int s_tiles, int s_splits, int s_chunk, int o_splits, int o_chunk,
    float* ws) {
  using S = typename Elem<T>::S;
  __shared__ StreamLds<D, R> lds;
  const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  const int group = a.heads / a.kv_heads, hs_n = a.n_seq * a.kv_heads;
  const int64_t all = (int64_t)hs_n * rows;
  const int front = a.kv_heads * s_tiles * s_splits;
  if ((int)blockIdx.x < front) {
    float2* ml = reinterpret_cast<float2*>(ws + s_splits * all * D);
    const int kh = blockIdx.x % a.kv_heads, rest = blockIdx.x / a.kv_heads;
    const int tile = rest % s_tiles, split = rest / s_tiles;
    s16x8_t qf[R][D / 16];
    int dst[R];
    int seen[R], p[R], at[R];
#pragma unroll
    for (int g = 0; g < R; ++g) {
      const int m = (tile * R + g) * 32 + c;  // up to 2^25
      const int seq = min(m / rows, a.n_seq - 1), r = m % rows;
      AttnSeq s = attn_seq(a, seq);
      int t = r / group;
      at[g] = kh * group + r % group;
      const bool live = m < a.n_seq * rows && t < s.nq;
      dst[g] = live ? (seq * a.kv_heads + kh) * rows + r : -1;  // up to 2^25
      seen[g] = sh.rows;
      p[g] = t + s.nk - s.nq + sh.rows;
      if (!live) s.q_at = 0, t = 0;  // a row that is there
      attn_load_q<T, D>(a, s, t, at[g], h, qf[g]);
    }
    AttnScore<kCap, kSlope> score[R];
    int near = INT_MAX;
#pragma unroll
    for (int g = 0; g < R; ++g) {
      score[g] = AttnScore<kCap, kSlope>(a, at[g]);
      near = min(near, dst[g] < 0 ? INT_MAX : p[g] + 1);
    }
    if constexpr (kSlope) {  // of all rows
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) near = min(near, __shfl_xor(near, off, 64));
      near = __builtin_amdgcn_readfirstlane(near);
    }
    const int begin = split * s_chunk;
    const StreamKeys keys{static_cast<const char*>(sh.k) + kh * sh.k_head * 2,
                          static_cast<const char*>(sh.v) + kh * sh.v_head * 2, sh.k_row * 2, sh.v_row * 2,
                          sh.rows};
    attn_stream<T, D, R, R, kCap, kSlope>(a, lds, keys, begin, min(sh.rows, begin + s_chunk), qf, score, seen,
                                       sh.rows, p, near, dst, ws + split * all * D, ml + split * all);
    return;
  }
  const int own = blockIdx.x - front, hs = own % hs_n, split = own / hs_n;
  const int kh = hs % a.kv_heads;
  const AttnSeq s = attn_seq(a, hs / a.kv_heads);
  const int live = s.nq * group;
  if (live == 0) return;
  const int m = min(c, live - 1), t = m / group, head = kh * group + m % group;
  const int seen[1] = {attn_seen(a, s, t)}, p[1] = {t + s.nk - s.nq};
  const int seen_hi = __builtin_amdgcn_readfirstlane(attn_seen(a, s, s.nq - 1));
  const int seen_lo = __builtin_amdgcn_readfirstlane(attn_seen(a, s, 0));
  const int begin = split * o_chunk, end = min(seen_hi, begin + o_chunk);
  if (begin >= end) return;  // the join reads the ranges up to seen_hi only
  s16x8_t qf[1][D / 16];
  attn_load_q<T, D>(a, s, t, head, h, qf[0]);
  const AttnScore<kCap, kSlope> score[1] = {AttnScore<kCap, kSlope>(a, head)};
  const int dst[1] = {c < live ? hs * rows + c : -1};
  // Keys below `near` are at or before every row's p, or hidden behind it.
  const int near = a.causal && !a.prefix_lens ? INT_MAX : s.nk - s.nq + 1;
  const StreamKeys keys{
      reinterpret_cast<const char*>(static_cast<const S*>(a.k) + s.k_at + kh * a.k_head),
      reinterpret_cast<const char*>(static_cast<const S*>(a.v) + s.v_at + kh * a.v_head), a.k_row * 2,
      a.v_row * 2, s.nk};
  ws += s_splits * all * (D + 2);
  float2* ml = reinterpret_cast<float2*>(ws + o_splits * all * D);
  attn_stream<T, D, 1, R, kCap, kSlope>(a, lds, keys, begin, end, qf, score, seen, seen_lo, p, near, dst,
                                        ws + split * all * D, ml + split * all);
}

// ---- any alignment and head dim: a wave a row, from the definition

template <int T, bool kCap, bool kSlope>
__global__ __launch_bounds__(256) void attn_shared_rows_kernel(AttnArgs a, AttnShared sh) {
  __shared__ float qs[4][256];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t items = (int64_t)a.n_seq * a.max_q * a.heads;
  for (int64_t item = (int64_t)blockIdx.x * 4 + wave; item < items; item += (int64_t)gridDim.x * 4) {
    const int head = (int)(item % a.heads);
    const int64_t row = item / a.heads;
    const int t = (int)(row % a.max_q);
    const AttnSeq s = attn_seq(a, (int)(row / a.max_q));
    if (t >= s.nq) continue;
    attn_row_shared<T, kCap, kSlope, unsigned>(a, sh, s, head, t, attn_seen(a, s, t), qs[wave]);
  }
}

// ---- launches

// Up to kJoinFew ranges 16 lanes a row take them all, four at a time; more are shared by 256.
constexpr int kJoinFew = 8;
template <int T, int D, bool kCap, bool kSlope>
void launch_shared_join(const AttnArgs& a, const AttnShared& sh, const AttnFront& front, int tile_rows,
                        int tiles, int64_t all, int splits, int chunk, int own0, const float* ws,
                        hipStream_t stream) {
  const AttnJoinShared before{sh, front, own0};
  if (front.ranges + splits > kJoinFew)
    hipLaunchKernelGGL((attn_shared_join_kernel<T, D, 16, kCap, kSlope>), dim3((unsigned)all), dim3(256),
                       0, stream, a, tile_rows, tiles, splits, chunk, ws, before);
  else
    hipLaunchKernelGGL((attn_shared_join_kernel<T, D, 1, kCap, kSlope>),
                       dim3((unsigned)((all + 15) / 16)), dim3(256), 0, stream, a, tile_rows, tiles, splits, chunk,
                       ws, before);
}

template <int T, int D, int R, bool kCap, bool kSlope>
hipError_t launch_stream(const AttnArgs& a, const AttnShared& sh, const SharedPlan& p, float* ws,
                         hipStream_t stream) {
  const int rows = a.max_q * (a.heads / a.kv_heads);
  const int64_t hs = (int64_t)a.n_seq * a.kv_heads;
  const unsigned blocks = (unsigned)((int64_t)a.kv_heads * p.s_tiles * p.s_splits + hs * p.o_splits);
  hipLaunchKernelGGL((attn_stream_kernel<T, D, R, kCap, kSlope>), dim3(blocks), dim3(kFewWaves * 64), 0,
                     stream, a, sh, rows, p.s_tiles, p.s_splits, p.s_chunk, p.o_splits, p.o_chunk, ws);
  launch_shared_join<T, D, kCap, kSlope>(a, sh, AttnFront{ws, hs * rows, p.s_splits, 0}, rows, 1, hs * rows,
                                         p.o_splits, p.o_chunk, 0, ws + p.s_splits * hs * rows * (D + 2), stream);
  return hipGetLastError();
}

// Sequences that fill little of their tiles: first all rows as they stand in q, one sequence, against
// ranges of the shared keys, then each sequence's against its own, on from those sums.
template <int T, int D, int WM, bool kCap>
hipError_t launch_packed(const AttnArgs& a, const AttnShared& sh, const SharedPlan& p, float* ws,
                         hipStream_t stream) {
  constexpr int kRows = WM * 32;
  AttnArgs f = a;  // one sequence of all rows
  f.k = sh.k, f.k_row = sh.k_row, f.k_head = sh.k_head;
  f.v = sh.v, f.v_row = sh.v_row, f.v_head = sh.v_head;
  f.k_seq = f.v_seq = f.q_seq = f.out_seq = 0;
  f.q_offsets = f.k_offsets = f.q_lens = f.k_lens = f.prefix_lens = nullptr;
  f.n_seq = 1, f.max_q = a.q_offsets ? a.q_rows : a.n_seq * a.max_q, f.max_k = sh.rows, f.causal = 0;
  const int group = a.heads / a.kv_heads;
  const int o_tiles = (a.max_q * group + kRows - 1) / kRows;
  const int64_t f_all = (int64_t)a.kv_heads * p.s_tiles * kRows;
  const dim3 block(attn_waves(WM) * 64);
  hipLaunchKernelGGL((attn_tiles_kernel<T, D, WM, kCap, false, true>),
                     dim3((unsigned)((int64_t)a.kv_heads * p.s_tiles * p.s_splits)), block, 0, stream, f,
                     p.s_tiles, p.s_tiles, 1, p.s_splits, p.s_chunk, ws);
  hipLaunchKernelGGL((attn_walk_kernel<T, D, WM, kCap, false, false, AttnSums>),
                     dim3((unsigned)((int64_t)a.n_seq * a.kv_heads * o_tiles)), block, 0, stream, a, o_tiles,
                     o_tiles, a.n_seq * a.kv_heads, 1, 0, nullptr,
                     AttnSums{sh, AttnFront{ws, f_all, p.s_splits, p.s_tiles * kRows}});
  return hipGetLastError();
}

template <int T, int D, int WM, bool kCap, bool kSlope>
hipError_t launch_shared_tiles(const AttnArgs& a, const AttnShared& sh, const AttnPlan& plan, int own0, float* ws,
                               hipStream_t stream) {
  constexpr int kRows = WM * 32;
  const int64_t rows = (int64_t)a.max_q * (a.heads / a.kv_heads);
  const int tiles = (int)((rows + kRows - 1) / kRows);
  const int64_t blocks = (int64_t)a.n_seq * a.kv_heads * tiles;
  const dim3 block(attn_waves(WM) * 64);
  if (plan.splits > 1) {
    hipLaunchKernelGGL((attn_walk_kernel<T, D, WM, kCap, kSlope, true, AttnShared>),
                       dim3((unsigned)(blocks * plan.splits)), block, 0, stream, a, tiles, plan.first, 1,
                       plan.splits, plan.chunk, ws, sh);
    launch_shared_join<T, D, kCap, kSlope>(a, sh, AttnFront{ws, 0, 0, 0}, kRows, tiles, blocks * kRows,
                                           plan.splits, plan.chunk, own0, ws, stream);
    return hipGetLastError();
  }
  hipLaunchKernelGGL((attn_walk_kernel<T, D, WM, kCap, kSlope, false, AttnShared>), dim3((unsigned)blocks), block,
                     0, stream, a, tiles, plan.first, plan.near_hs, 1, 0, nullptr, sh);
  return hipGetLastError();
}

template <int T, bool kCap, bool kSlope>
hipError_t launch_shared_scored(const AttnArgs& a, const AttnShared& sh, const SharedPlan& p, float* ws,
                                hipStream_t stream) {
  const bool wide = a.dim > 64;
  switch (p.kernel) {
    case IMQ_SHARED_ROWS: {
      const int64_t blocks = ((int64_t)a.n_seq * a.max_q * a.heads + 3) / 4;
      const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)));
      hipLaunchKernelGGL((attn_shared_rows_kernel<T, kCap, kSlope>), grid, dim3(256), 0, stream, a, sh);
      return hipGetLastError();
    }
    case IMQ_SHARED_STREAM:
      if (p.s_rows == 64)
        return wide ? launch_stream<T, 128, 2, kCap, kSlope>(a, sh, p, ws, stream)
                    : launch_stream<T, 64, 2, kCap, kSlope>(a, sh, p, ws, stream);
      return wide ? launch_stream<T, 128, 1, kCap, kSlope>(a, sh, p, ws, stream)
                  : launch_stream<T, 64, 1, kCap, kSlope>(a, sh, p, ws, stream);
    case IMQ_SHARED_PACKED:
      if constexpr (!kSlope)
        return wide ? launch_packed<T, 128, 4, kCap>(a, sh, p, ws, stream)
                    : launch_packed<T, 64, 4, kCap>(a, sh, p, ws, stream);
      return hipErrorInvalidValue;
    default: break;
  }
  switch (wide ? p.tiles.tile_rows : -p.tiles.tile_rows) {
    case 128: return launch_shared_tiles<T, 128, 4, kCap, kSlope>(a, sh, p.tiles, p.own0, ws, stream);
    case 64: return launch_shared_tiles<T, 128, 2, kCap, kSlope>(a, sh, p.tiles, p.own0, ws, stream);
    case -128: return launch_shared_tiles<T, 64, 4, kCap, kSlope>(a, sh, p.tiles, p.own0, ws, stream);
    case -64: return launch_shared_tiles<T, 64, 2, kCap, kSlope>(a, sh, p.tiles, p.own0, ws, stream);
    default: return hipErrorInvalidValue;
  }
}

template <int T>
hipError_t launch_shared_t(const AttnArgs& a, const AttnShared& sh, const SharedPlan& p, float* ws,
                           hipStream_t stream) {
  const bool cap = a.softcap > 0.f, slope = a.slopes != nullptr;
  if (cap && slope) return launch_shared_scored<T, true, true>(a, sh, p, ws, stream);
  if (cap) return launch_shared_scored<T, true, false>(a, sh, p, ws, stream);
  if (slope) return launch_shared_scored<T, false, true>(a, sh, p, ws, stream);
  return launch_shared_scored<T, false, false>(a, sh, p, ws, stream);
}

}  // namespace imq
