// core.cpp -- the C entry points of include/imq_core.h: argument checks, the
// attention's plan and workspace, and the launches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <utility>

#include "core_kernels.hpp"
#include "ctx.hpp"
#include "imq.h"
#include "imq_core.h"

using namespace imq::detail;

namespace {

bool known(imq_dtype t) { return t == IMQ_BF16 || t == IMQ_F16 || t == IMQ_F32; }

// The largest element offset of a tensor walked by these extents and strides,
// or -1 where a stride is negative or the bytes pass 2^62.
int64_t reach(std::initializer_list<std::pair<int64_t, int64_t>> extents) {
  __int128 at = 0;
  for (const auto& e : extents) {
    if (e.second < 0) return -1;
    at += (__int128)(e.first > 0 ? e.first - 1 : 0) * e.second;
  }
  return at < ((__int128)1 << 60) ? (int64_t)at : -1;
}

// Whether two of the places that these extents and strides give, `dim` elements each,
// lie on each other.  Strides that fit into each other do not, in any order; of others
// every difference of two places is looked at, as far as 2^20 steps go (then: yes).
// (Their reach has been checked: sums stay under 2^61.)
using Extent = std::pair<int64_t, int64_t>;
inline bool nested(int64_t dim, const Extent* e, int n) {
  int64_t span = dim;
  bool fit = true;
  for (int i = 0; i < n; ++i)
    if (e[i].first > 1) {
      fit = fit && e[i].second >= span;
      span += (e[i].first - 1) * e[i].second;
    }
  return fit;
}

bool on_each_other_slow(int64_t dim, const Extent* extents, int count) {
  Extent e[3];  // (extent, stride) of those that step, strides rising
  int n = 0;
  for (int i = 0; i < count; ++i)
    if (extents[i].first > 1) e[n++] = extents[i];
  std::sort(e, e + n, [](const auto& a, const auto& b) { return a.second < b.second; });
  if (nested(dim, e, n)) return false;
  // The longest is solved for, the others are stepped through (both signs of one do).
  std::sort(e, e + n, [](const auto& a, const auto& b) { return a.first > b.first; });
  const int64_t n1 = n > 1 ? e[1].first : 1, n2 = n > 2 ? e[2].first : 1, s0 = e[0].second;
  if (s0 < dim || (__int128)(2 * n1 - 1) * n2 > (1 << 20)) return true;
  for (int64_t c = 0; c < n2; ++c)
    for (int64_t b = c == 0 ? 0 : 1 - n1; b < n1; ++b) {
      __int128 at = 0;
      if (n > 1) at += (__int128)b * e[1].second;
      if (n > 2) at += (__int128)c * e[2].second;
      // The two multiples of s0 next to `at`.
      const __int128 low = at >= 0 ? at / s0 : -((-at + s0 - 1) / s0);
      for (__int128 a = low; a <= low + 1; ++a) {
        if (a >= e[0].first || a <= -e[0].first || (a == 0 && b == 0 && c == 0)) continue;
        const __int128 away = at - a * s0;
        if (away < dim && -away < dim) return true;
      }
    }
  return false;
}

// Mostly they rise as they are given: nothing is sorted then.
template <int N>
bool on_each_other(int64_t dim, const Extent (&e)[N]) {
  return !nested(dim, e, N) && on_each_other_slow(dim, e, N);
}

int check_attention(imq_ctx* ctx, const char* fn, const imq_attention_args* p, imq::AttnArgs* a) {
  if (!ctx) return fail(nullptr, IMQ_EINVAL, "%s: null context", fn);
  if (!p) return fail(ctx, IMQ_EINVAL, "%s: null arguments", fn);
  if (p->dtype != IMQ_BF16 && p->dtype != IMQ_F16)
    return fail(ctx, IMQ_EUNSUPPORTED, "%s: dtype %d (bf16 and f16 are provided)", fn,
                p->dtype);
  if (p->n_seq < 0 || p->max_q < 0 || p->max_k < 0 || p->q_rows < 0 || p->k_rows < 0)
    return fail(ctx, IMQ_EINVAL, "%s: n_seq %d, max_q %d, max_k %d, q_rows %d, k_rows %d", fn,
                p->n_seq, p->max_q, p->max_k, p->q_rows, p->k_rows);
  if (p->heads <= 0 || p->kv_heads <= 0 || p->heads % p->kv_heads != 0)
    return fail(ctx, IMQ_EINVAL, "%s: %d heads are not whole groups of %d key heads", fn, p->heads,
                p->kv_heads);
  if (p->dim <= 0) return fail(ctx, IMQ_EINVAL, "%s: head dim %d", fn, p->dim);
  if (p->dim > 256)
    return fail(ctx, IMQ_EUNSUPPORTED, "%s: head dim %d (1 to 256 are provided)", fn, p->dim);
  if (!std::isfinite(p->scale) || p->scale <= 0.f)
    return fail(ctx, IMQ_EINVAL, "%s: scale %g must be finite and positive", fn, (double)p->scale);
  if (!std::isfinite(p->softcap) || p->softcap < 0.f)
    return fail(ctx, IMQ_EINVAL, "%s: softcap %g must be finite and not negative", fn,
                (double)p->softcap);
  // A capped score is a difference of numbers of the cap's size.
  if (p->softcap > 4096.f)
    return fail(ctx, IMQ_EUNSUPPORTED, "%s: softcap %g (up to 4096)", fn, (double)p->softcap);
  if (!std::isfinite((p->softcap > 0.f ? 2.f * p->scale / p->softcap : p->scale) * 1.5f))
    return fail(ctx, IMQ_EINVAL, "%s: scale %g over softcap %g leaves fp32", fn, (double)p->scale,
                (double)p->softcap);
  // Within a tile, what a slope takes is divided by the scale (attn_start, attn_scores):
  // 2^20 a key over 2^30 keys, over 2^-64, stays in fp32.
  if (p->slopes && p->softcap == 0.f && p->scale < 0x1p-64f)
    return fail(ctx, IMQ_EUNSUPPORTED, "%s: scale %g with slopes (2^-64 and above)", fn, (double)p->scale);
  if (p->causal != 0 && p->causal != 1)
    return fail(ctx, IMQ_EINVAL, "%s: causal %d (0 or 1)", fn, p->causal);
  if (p->prefix_lens && !p->causal)
    return fail(ctx, IMQ_EINVAL, "%s: prefix_lens without causal", fn);
  if (p->q_offsets && p->q_lens)
    return fail(ctx, IMQ_EINVAL, "%s: q_offsets and q_lens exclude each other", fn);
  if (p->k_offsets && p->k_lens)
    return fail(ctx, IMQ_EINVAL, "%s: k_offsets and k_lens exclude each other", fn);
  const int64_t qs = p->q_offsets ? 0 : p->q_seq, ks = p->k_offsets ? 0 : p->k_seq;
  const int64_t vs = p->k_offsets ? 0 : p->v_seq, os = p->q_offsets ? 0 : p->out_seq;
  const int64_t qr = p->q_offsets ? p->q_rows : p->max_q, kr = p->k_offsets ? p->k_rows : p->max_k;
  if (reach({{p->n_seq, qs}, {qr, p->q_row}, {p->heads, p->q_head}}) < 0 ||
      reach({{p->n_seq, ks}, {kr, p->k_row}, {p->kv_heads, p->k_head}}) < 0 ||
      reach({{p->n_seq, vs}, {kr, p->v_row}, {p->kv_heads, p->v_head}}) < 0 ||
      reach({{p->n_seq, os}, {qr, p->out_row}, {p->heads, p->out_head}}) < 0)
    return fail(ctx, IMQ_EINVAL, "%s: a negative stride, or a tensor past 2^60 elements", fn);
  // Outputs that lie on each other: two rows, heads or sequences at one place.
  // (Lengths may keep sequences apart that reach into each other's windows.)
  const int64_t apart = p->q_offsets || p->q_lens ? 1 : p->n_seq;
  if ((p->heads > 1 && p->out_head < p->dim) || (qr > 1 && p->out_row < p->dim) ||
      (!p->q_offsets && p->n_seq > 1 && p->out_seq < p->dim) ||
      on_each_other(p->dim, {{p->heads, p->out_head}, {qr, p->out_row}, {apart, os}}))
    return fail(ctx, IMQ_EINVAL, "%s: out's strides (%lld, %lld, %lld) lay outputs on each other", fn,
                (long long)p->out_seq, (long long)p->out_row, (long long)p->out_head);
  if (p->n_seq > 0 && p->max_q > 0) {
    if (!p->q || !p->out || (p->max_k > 0 && (!p->k || !p->v)))
      return fail(ctx, IMQ_EINVAL, "%s: null device pointer (q=%p k=%p v=%p out=%p)", fn, p->q, p->k,
                  p->v, p->out);
    if (p->out == p->q || (p->max_k > 0 && (p->out == p->k || p->out == p->v)))
      return fail(ctx, IMQ_EINVAL, "%s: out is q, k or v", fn);
    if (!aligned(p->q, 2) || !aligned(p->k, 2) || !aligned(p->v, 2) || !aligned(p->out, 2))
      return fail(ctx, IMQ_EINVAL, "%s: q, k, v and out must be 2-byte aligned", fn);
  }
  for (const void* d : {(const void*)p->q_offsets, (const void*)p->k_offsets, (const void*)p->q_lens,
                        (const void*)p->k_lens, (const void*)p->prefix_lens, (const void*)p->slopes})
    if (!aligned(d, 4))
      return fail(ctx, IMQ_EINVAL, "%s: offsets, lengths and slopes must be 4-byte aligned", fn);
  a->q = p->q, a->k = p->k, a->v = p->v, a->out = p->out;
  a->q_seq = qs, a->q_row = p->q_row, a->q_head = p->q_head;
  a->k_seq = ks, a->k_row = p->k_row, a->k_head = p->k_head;
  a->v_seq = vs, a->v_row = p->v_row, a->v_head = p->v_head;
  a->out_seq = os, a->out_row = p->out_row, a->out_head = p->out_head;
  a->q_offsets = p->q_offsets, a->k_offsets = p->k_offsets;
  a->q_lens = p->q_lens, a->k_lens = p->k_lens, a->prefix_lens = p->prefix_lens;
  a->slopes = p->slopes;
  a->n_seq = p->n_seq, a->heads = p->heads, a->kv_heads = p->kv_heads, a->dim = p->dim;
  // A packed sequence is no longer than all of its rows.
  a->max_q = p->q_offsets ? std::min(p->max_q, p->q_rows) : p->max_q;
  a->max_k = p->k_offsets ? std::min(p->max_k, p->k_rows) : p->max_k;
  a->q_rows = p->q_rows, a->k_rows = p->k_rows;
  a->causal = p->causal, a->scale = p->scale, a->softcap = p->softcap;
  return IMQ_OK;
}

}  // namespace

extern "C" {

int imq_ln_mod(imq_ctx* ctx, const void* x, imq_dtype x_dtype, const float* shift,
               const float* scale, const int32_t* sets, int n_sets, void* y, imq_dtype y_dtype,
               int rows, int cols, float eps, float post, imq_stream stream) {
  const char* fn = "imq_ln_mod";
  if (!ctx) return fail(nullptr, IMQ_EINVAL, "%s: null context", fn);
  if (y_dtype != IMQ_BF16 && y_dtype != IMQ_F16)
    return fail(ctx, IMQ_EUNSUPPORTED, "%s: y dtype %d (bf16 or f16)", fn, (int)y_dtype);
  if (x_dtype != IMQ_F32 && x_dtype != y_dtype)
    return fail(ctx, IMQ_EUNSUPPORTED, "%s: x dtype %d (f32, or y's dtype)", fn, (int)x_dtype);
  if (rows < 0 || cols <= 0 || n_sets <= 0)
    return fail(ctx, IMQ_EINVAL, "%s: rows %d, cols %d, n_sets %d", fn, rows, cols, n_sets);
  // The sums are 256 threads' in fp32: 2^12 terms each are right to 2^-12.
  if (cols > 1 << 20) return fail(ctx, IMQ_EUNSUPPORTED, "%s: %d columns (up to 2^20)", fn, cols);
  if (!sets && n_sets != 1)
    return fail(ctx, IMQ_EINVAL, "%s: %d modulations without sets", fn, n_sets);
  if (!std::isfinite(eps) || eps < 0.f)
    return fail(ctx, IMQ_EINVAL, "%s: eps %g must be finite and non-negative", fn, (double)eps);
  if (!std::isfinite(post))
    return fail(ctx, IMQ_EINVAL, "%s: post %g must be finite", fn, (double)post);
  if (rows == 0) return IMQ_OK;
  if (!x || !shift || !scale || !y) return fail(ctx, IMQ_EINVAL, "%s: null device pointer", fn);
  if (!aligned(x, elem_size(x_dtype)) || !aligned(shift, 4) || !aligned(scale, 4) ||
      !aligned(sets, 4) || !aligned(y, 2))
    return fail(ctx, IMQ_EINVAL, "%s: x, shift, scale, sets or y misaligned for its element type",
                fn);
  if (x == y && x_dtype != y_dtype)
    return fail(ctx, IMQ_EINVAL, "%s: in place needs x and y of one type", fn);
  int rc = bind_device(ctx);
  if (rc != IMQ_OK) return rc;
  const hipError_t e = imq::launch_ln_mod(x, (int)x_dtype, shift, scale, sets, n_sets, y,
                                          (int)y_dtype, rows, cols, eps, post,
                                          static_cast<hipStream_t>(stream));
  return e == hipSuccess ? IMQ_OK : hip_fail(ctx, e, fn);
}

int imq_rope(imq_ctx* ctx, const imq_rope_heads* groups, int n_groups, int rows, int dim,
             int rot_dim, int interleaved, const int32_t* positions, int axes, const int* sections,
             const double* inv_freq, float amplitude, float eps, imq_dtype dtype,
             imq_stream stream) {
  const char* fn = "imq_rope";
  if (!ctx) return fail(nullptr, IMQ_EINVAL, "%s: null context", fn);
  if (!known(dtype))
    return fail(ctx, IMQ_EUNSUPPORTED, "%s: dtype %d (bf16, f16 and f32 are provided)", fn,
                (int)dtype);
  if (!groups || n_groups < 1 || n_groups > 2)
    return fail(ctx, IMQ_EINVAL, "%s: %d groups of heads (1 or 2)", fn, n_groups);
  if (dim > 1024) return fail(ctx, IMQ_EUNSUPPORTED, "%s: head dim %d (up to 1024)", fn, dim);
  if (rows < 0 || dim < 2 || dim % 2 != 0 || rot_dim < 0 || rot_dim > dim || rot_dim % 2 != 0)
    return fail(ctx, IMQ_EINVAL, "%s: rows %d, head dim %d, rotated %d", fn, rows, dim, rot_dim);
  if (interleaved != 0 && interleaved != 1)
    return fail(ctx, IMQ_EINVAL, "%s: interleaved %d (0 or 1)", fn, interleaved);
  if (!std::isfinite(eps) || eps < 0.f || !std::isfinite(amplitude))
    return fail(ctx, IMQ_EINVAL, "%s: eps %g must be finite and not negative, amplitude %g finite",
                fn, (double)eps, (double)amplitude);
  if (axes < 1 || axes > 4 || (!sections && axes != 1))
    return fail(ctx, IMQ_EINVAL, "%s: %d axes (1 to 4; more than one with sections)", fn, axes);
  imq::RopeArgs a{};
  int at = 0;
  for (int i = 0; i < 4; ++i) {
    if (i < axes && sections) {
      if (sections[i] < 0 || sections[i] > rot_dim / 2)
        return fail(ctx, IMQ_EINVAL, "%s: section %d has %d pairs", fn, i, sections[i]);
      at += sections[i];
    }
    a.section_end[i] = sections ? at : rot_dim / 2;
  }
  if (sections && at != rot_dim / 2)
    return fail(ctx, IMQ_EINVAL, "%s: the sections hold %d pairs of %d", fn, at, rot_dim / 2);
  if (rows > 0 && rot_dim > 0 && (!positions || !inv_freq))
    return fail(ctx, IMQ_EINVAL, "%s: null positions or inv_freq", fn);
  if (!aligned(positions, 4) || !aligned(inv_freq, 8))
    return fail(ctx, IMQ_EINVAL, "%s: positions must be 4-byte, inv_freq 8-byte aligned", fn);
  const size_t es = elem_size(dtype);
  for (int i = 0; i < n_groups; ++i) {
    const imq_rope_heads& g = groups[i];
    if (g.heads < 0) return fail(ctx, IMQ_EINVAL, "%s: group %d has %d heads", fn, i, g.heads);
    if (reach({{rows, g.x_row}, {g.heads, g.x_head}}) < 0 ||
        reach({{rows, g.y_row}, {g.heads, g.y_head}}) < 0)
      return fail(ctx, IMQ_EINVAL, "%s: group %d: a negative stride, or a tensor past 2^60 elements",
                  fn, i);
    if ((g.heads > 1 && g.y_head < dim) || (rows > 1 && g.y_row < dim) ||
        on_each_other(dim, {{g.heads, g.y_head}, {rows, g.y_row}}))
      return fail(ctx, IMQ_EINVAL, "%s: group %d: y's strides (%lld, %lld) lay outputs on each other",
                  fn, i, (long long)g.y_row, (long long)g.y_head);
    if (rows > 0 && g.heads > 0) {
      if (!g.x || !g.y) return fail(ctx, IMQ_EINVAL, "%s: group %d: null device pointer", fn, i);
      if (!aligned(g.x, es) || !aligned(g.y, es) || !aligned(g.weight, 4))
        return fail(ctx, IMQ_EINVAL, "%s: group %d: x, y or weight misaligned for its element type",
                    fn, i);
      if (g.x == g.y && (g.x_row != g.y_row || g.x_head != g.y_head))
        return fail(ctx, IMQ_EINVAL, "%s: group %d: in place needs equal strides", fn, i);
    }
    a.g[i] = imq::RopeGroup{g.x, g.y, g.weight, g.x_row, g.x_head, g.y_row, g.y_head, g.heads};
  }
  a.positions = positions, a.inv_freq = inv_freq;
  a.groups = n_groups, a.rows = rows, a.dim = dim, a.rot = rot_dim, a.axes = axes;
  a.amplitude = amplitude, a.eps = eps;
  int rc = bind_device(ctx);
  if (rc != IMQ_OK) return rc;
  const hipError_t e =
      imq::launch_rope(a, interleaved != 0, (int)dtype, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? IMQ_OK : hip_fail(ctx, e, fn);
}

int imq_attention(imq_ctx* ctx, const imq_attention_args* args, imq_stream stream) {
  const char* fn = "imq_attention";
  imq::AttnArgs a{};
  int rc = check_attention(ctx, fn, args, &a);
  if (rc != IMQ_OK) return rc;
  if (a.n_seq == 0 || a.max_q == 0) return IMQ_OK;
  if ((rc = bind_device(ctx)) != IMQ_OK) return rc;
  const auto st = static_cast<hipStream_t>(stream);
  imq::AttnPlan plan = imq::attention_plan(a, ctx->cus);
  SplitHold hold;  // until the join is enqueued
  if (plan.bytes > 0) {
    hold = split_ws(ctx, st, plan.bytes);
    if (!hold.ws.p) {  // it would have to grow under capture, or memory is short
      plan.splits = 1;
      plan.bytes = 0;
    }
  }
  const hipError_t e = imq::launch_attention(a, plan, hold.ws.p, args->dtype, st);
  return e == hipSuccess ? IMQ_OK : hip_fail(ctx, e, fn);
}

int imq_attention_plan(imq_ctx* ctx, const imq_attention_args* args, imq_attention_plan_info* out) {
  const char* fn = "imq_attention_plan";
  imq::AttnArgs a{};
  const int rc = check_attention(ctx, fn, args, &a);
  if (rc != IMQ_OK) return rc;
  if (!out) return fail(ctx, IMQ_EINVAL, "%s: null output", fn);
  const imq::AttnPlan p = imq::attention_plan(a, ctx->cus);
  out->kernel = p.kernel;
  out->tile_rows = p.tile_rows;
  out->splits = p.splits;
  out->workspace_bytes = p.bytes;
  return IMQ_OK;
}

}  // extern "C"
