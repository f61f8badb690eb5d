// attention.hpp -- device code shared by the attention kernels: where a
// sequence's rows are, what a query sees, how a score becomes an exponent of
// two, and one query's output by a whole wave.
#pragma once

#include <climits>

#include "core_kernels.hpp"
#include "imq_device.hpp"

namespace imq {

constexpr float kLog2e = 1.44269504088896340736f;

// The rows of one sequence.  Lengths and offsets come from device memory and
// are clamped to what the tensors hold.
struct AttnSeq {
  int64_t q_at, k_at, v_at, out_at;  // element offsets of row 0, head 0
  int nq, nk, prefix;
};

__device__ __forceinline__ AttnSeq attn_seq(const AttnArgs& a, int s) {
  AttnSeq r;
  if (a.q_offsets) {
    const int b = min(max(a.q_offsets[s], 0), a.q_rows);
    const int e = min(max(a.q_offsets[s + 1], b), a.q_rows);
    r.nq = min(e - b, a.max_q);
    r.q_at = b * a.q_row;
    r.out_at = b * a.out_row;
  } else {
    r.nq = a.q_lens ? min(max(a.q_lens[s], 0), a.max_q) : a.max_q;
    r.q_at = s * a.q_seq;
    r.out_at = s * a.out_seq;
  }
  if (a.k_offsets) {
    const int b = min(max(a.k_offsets[s], 0), a.k_rows);
    const int e = min(max(a.k_offsets[s + 1], b), a.k_rows);
    r.nk = min(e - b, a.max_k);
    r.k_at = b * a.k_row;
    r.v_at = b * a.v_row;
  } else {
    r.nk = a.k_lens ? min(max(a.k_lens[s], 0), a.max_k) : a.max_k;
    r.k_at = s * a.k_seq;
    r.v_at = s * a.v_seq;
  }
  r.prefix = a.prefix_lens ? min(max(a.prefix_lens[s], 0), r.nk) : 0;
  return r;
}

// Query t sees the keys [0, attn_seen): every mask here leaves one range.
__device__ __forceinline__ int attn_seen(const AttnArgs& a, const AttnSeq& s, int t) {
  if (!a.causal) return s.nk;
  return max(min(max(t + s.nk - s.nq + 1, 0), s.nk), s.prefix);
}

// e = score(q . k, |p - j|) in units of log2: the softmax runs on v_exp_f32,
// which is a power of two.  tanh(z) = 1 - 2 / (exp(2 z) + 1) is exact to a few
// 2^-24 absolutely and has its limits at infinite arguments.
template <bool kCap, bool kSlope>
struct AttnScore {
  float mul;   // scale * log2(e), or 2 * scale / cap * log2(e)
  float top;   // cap * log2(e)
  float fall;  // slope * log2(e)

  AttnScore() = default;
  __device__ __forceinline__ AttnScore(const AttnArgs& a, int head) {
    mul = kCap ? 2.f * a.scale / a.softcap * kLog2e : a.scale * kLog2e;
    top = kCap ? a.softcap * kLog2e : 0.f;
    fall = kSlope ? a.slopes[head] * kLog2e : 0.f;
  }
  __device__ __forceinline__ float rest(float dot) const {
    return __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(dot * mul) + 1.f);
  }
  __device__ __forceinline__ float capped(float dot) const { return top - 2.f * top * rest(dot); }
  __device__ __forceinline__ float operator()(float dot, float away) const {
    float e = kCap ? capped(dot) : dot * mul;
    if constexpr (kSlope) e = __builtin_fmaf(-fall, __builtin_fabsf(away), e);
    return e;
  }
};

// One query's output by a whole wave, from the definition: 64 keys at a time,
// a key per lane for the scores, `dim` elements over the lanes for the product
// with v, the running maximum and sum rescaled per 64 keys.  Only keys below
// `seen` are read, so nothing that a mask hides can reach the output.
// qs: dim floats of LDS of this wave's own.  J counts the keys: unsigned where there may be more than
// 2^31 - 64 of them, past which the last step leaves an int.
template <int T, bool kCap, bool kSlope, class J = int>
__device__ void attn_row(const AttnArgs& a, const AttnSeq& s, int head, int t, int seen,
                         float* qs) {
  using S = typename Elem<T>::S;
  const int lane = threadIdx.x & 63;
  const int kh = head / (a.heads / a.kv_heads);
  const S* q = static_cast<const S*>(a.q) + s.q_at + t * a.q_row + head * a.q_head;
  const S* k = static_cast<const S*>(a.k) + s.k_at + kh * a.k_head;
  const S* v = static_cast<const S*>(a.v) + s.v_at + kh * a.v_head;
  S* out = static_cast<S*>(a.out) + s.out_at + t * a.out_row + head * a.out_head;
  const AttnScore<kCap, kSlope> score(a, head);
  for (int d = lane; d < a.dim; d += 64) qs[d] = Elem<T>::param(q[d]);
  __builtin_amdgcn_wave_barrier();
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, top = -INFINITY, sum = 0.f;
  const int p = t + s.nk - s.nq;
  for (J at = 0; at < (J)seen; at += 64) {
    const int j0 = (int)at, j = j0 + lane;
    float e = -INFINITY;
    if (j < seen) {
      const S* kr = k + (int64_t)j * a.k_row;
      float dot = 0.f;
      for (int d = 0; d < a.dim; ++d) dot = __builtin_fmaf(qs[d], Elem<T>::param(kr[d]), dot);
      e = score(dot, (float)(p - j));
    }
    float m = e;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
    // fmaxf drops a NaN; the weight below brings it back into the sum.
    const float next = fmaxf(top, m);
    const float base = next == -INFINITY ? 0.f : next;
    const float keep = __builtin_amdgcn_exp2f(top - base);
    const float w = __builtin_amdgcn_exp2f(e - base);
    float ws = w;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) ws += __shfl_xor(ws, off, 64);
    sum = sum * keep + ws;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] *= keep;
    top = next;
    const int n = min(64, seen - j0);
    for (int i = 0; i < n; ++i) {
      const float wi = __builtin_bit_cast(
          float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), i));
      const S* vr = v + (int64_t)(j0 + i) * a.v_row;
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (lane + 64 * c < a.dim)
          acc[c] = __builtin_fmaf(wi, Elem<T>::param(vr[lane + 64 * c]), acc[c]);
    }
  }
  const float inv = seen > 0 ? 1.f / sum : 0.f;
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (lane + 64 * c < a.dim) {
      const float o = acc[c] * inv;
      out[lane + 64 * c] = (S)(Elem<T>::pack2(o, o) & 0xFFFFu);
    }
}

// The same where the keys `sh` come before the sequence's own and are all seen.
struct AttnRowSums {
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, top = -INFINITY, sum = 0.f;
};

// The first n keys at k and v (rows k_row and v_row apart), key j at p - j from the query.
// Weights are 2^-32 of what they are, so that the largest bf16 values of 2^32 keys add up in fp32.
template <int T, class J, bool kCap, bool kSlope>
__device__ __forceinline__ void attn_row_keys(const AttnArgs& a, const typename Elem<T>::S* k,
                                              const typename Elem<T>::S* v, int64_t k_row,
                                              int64_t v_row, int n_keys, int p,
                                              const AttnScore<kCap, kSlope>& score,
                                              const float* qs, AttnRowSums& r) {
  using S = typename Elem<T>::S;
  const int lane = threadIdx.x & 63;
  for (J at = 0; at < (J)n_keys; at += 64) {
    const int j0 = (int)at, j = j0 + lane;
    float e = -INFINITY;
    if (j < n_keys) {
      const S* kr = k + (int64_t)j * k_row;
      float dot = 0.f;
      for (int d = 0; d < a.dim; ++d) dot = __builtin_fmaf(qs[d], Elem<T>::param(kr[d]), dot);
      e = score(dot, (float)(p - j));
    }
    float m = e;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
    // fmaxf drops a NaN; the weight below brings it back into the sum.
    const float next = fmaxf(r.top, m);
    const float base = next == -INFINITY ? 0.f : next;
    const float keep = __builtin_amdgcn_exp2f(r.top - base);
    const float w = __builtin_amdgcn_exp2f(e - base) * 0x1p-32f;
    float ws = w;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) ws += __shfl_xor(ws, off, 64);
    r.sum = r.sum * keep + ws;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.acc[i] *= keep;
    r.top = next;
    const int n = min(64, n_keys - j0);
    for (int i = 0; i < n; ++i) {
      const float wi = __builtin_bit_cast(
          float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), i));
      const S* vr = v + (int64_t)(j0 + i) * v_row;
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (lane + 64 * c < a.dim)
          r.acc[c] = __builtin_fmaf(wi, Elem<T>::param(vr[lane + 64 * c]), r.acc[c]);
    }
  }
}

template <int T, bool kCap, bool kSlope, class J = int>
__device__ void attn_row_shared(const AttnArgs& a, const AttnShared& sh, const AttnSeq& s, int head, int t,
                                int seen, float* qs) {
  using S = typename Elem<T>::S;
  const int lane = threadIdx.x & 63;
  const int kh = head / (a.heads / a.kv_heads);
  const S* q = static_cast<const S*>(a.q) + s.q_at + t * a.q_row + head * a.q_head;
  const S* k = static_cast<const S*>(a.k) + s.k_at + kh * a.k_head;
  const S* v = static_cast<const S*>(a.v) + s.v_at + kh * a.v_head;
  S* out = static_cast<S*>(a.out) + s.out_at + t * a.out_row + head * a.out_head;
  const AttnScore<kCap, kSlope> score(a, head);
  for (int d = lane; d < a.dim; d += 64) qs[d] = Elem<T>::param(q[d]);
  __builtin_amdgcn_wave_barrier();
  AttnRowSums r;
  const int p = t + s.nk - s.nq;
  attn_row_keys<T, J>(a, static_cast<const S*>(sh.k) + kh * sh.k_head,
                   static_cast<const S*>(sh.v) + kh * sh.v_head, sh.k_row, sh.v_row, sh.rows, sh.rows + p,
                   score, qs, r);
  attn_row_keys<T, J>(a, k, v, a.k_row, a.v_row, seen, p, score, qs, r);
  const float inv = seen > 0 || sh.rows > 0 ? 1.f / r.sum : 0.f;
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (lane + 64 * c < a.dim) {
      const float o = r.acc[c] * inv;
      out[lane + 64 * c] = (S)(Elem<T>::pack2(o, o) & 0xFFFFu);
    }
}

// The kernel's arguments, its first parameter, read anew.  For what is hardly ever
// run: arguments that only it needs would take scalar registers from the rest (the
// join 4.0 us against 4.3, as others were read twice).
__device__ __forceinline__ AttnArgs attn_args_again() {
  typedef const __attribute__((address_space(4))) AttnArgs* P;
  P p = (P)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));  // not the same load to the compiler
  return *(const AttnArgs*)p;
}

// The last key of [from, to) whose value of key head kh holds a NaN or an infinity,
// below `from` where none does; a key a lane, the whole wave.
template <int T>
__device__ int attn_last_odd(const AttnArgs& a, const AttnSeq& s, int kh, int from, int to) {
  using S = typename Elem<T>::S;
  constexpr unsigned kExp = T == kBf16 ? 0x7F80u : 0x7C00u;
  const S* v = static_cast<const S*>(a.v) + s.v_at + kh * a.v_head;
  const int lane = threadIdx.x & 63;
  for (int end = to; end > from; end -= 64) {
    const int j = end - 1 - lane;
    bool odd = false;
    if (j >= from) {
      const S* vr = v + (int64_t)j * a.v_row;
      for (int d = 0; d < a.dim; ++d) odd = odd || (vr[d] & kExp) == kExp;
    }
    const uint64_t any = __builtin_amdgcn_ballot_w64(odd);
    if (any) return end - 1 - __builtin_ctzll(any);
  }
  return from - 1;
}

// Which outputs that are not finite are made again (attn_row).  A tile multiplies the
// values of the keys that it hides by a weight of zero, which a NaN or an infinity
// outlives; what a query sees is no cause to do so: its scores' NaN are in the sum of
// the weights (a hidden key's are not), and a NaN or an infinity among its values
// belongs into the output.  So a row is made again that has a finite sum and a key
// behind its own, among those that its tile went through, with such a value.  An
// overflow that every query sees would otherwise cost a wave a row: 16384 causal rows
// of 32 heads 1.2 s against 2 ms.
// walked: the keys that tiles went through, at least.
template <int T>
__device__ __forceinline__ int attn_spoilt(const AttnArgs& a, const AttnSeq& s, int kh, int seen,
                                           int walked) {
  // Rows of values that begin inside the row before: a tile reads parts of the last
  // ones behind them, in other columns.
  if (a.v_row < a.dim) return INT_MAX;
  return attn_last_odd<T>(a, s, kh, seen, min(walked, s.nk));
}

}  // namespace imq
