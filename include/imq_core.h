/*
 * imq_core.h -- what stands between the quantized projections of a block.
 *
 * The reference's direct engine runs, around the qmm calls that imq.h,
 * imq_te.h and imq_step.h replace, a LayerNorm with the block's modulation
 * (lnMod: dd_ln_mod_prescale, Sources/ImarelloDirect/DirectDiTKernels.swift:16-59),
 * per-head RMSNorm of the queries and keys (dd_rmsnorm_pitched :61-99,
 * dq_rmsnorm, DirectGlueKernels.swift:14-49), RoPE (dd_rope_interleaved,
 * DirectDiTKernels.swift:103-122; dq_rope, DirectGlueKernels.swift:54-75) and
 * softmax attention (steel_attention, DirectDiTStep.swift:457-488,
 * DirectTEEncoder.swift:159-202).  The three entry points here are that work:
 * with them a caller of the block halves (imq_step.h) and of the layer halves
 * (imq_te.h) runs whole blocks and layers.
 *
 * Conventions as in imq.h: an imq_status is returned, nothing throws, calls
 * are asynchronous on the given stream and may be captured into a graph,
 * inputs are never written (but where an output is said to be allowed to be
 * its input).  Strides count elements.  Device arrays of lengths, offsets and
 * positions are read when the kernel runs: values that the description does
 * not allow cannot be refused then, and are clamped so that no access leaves
 * the tensors that the arguments describe.
 */
#ifndef IMQ_CORE_H
#define IMQ_CORE_H

#include "imq.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- modulated LayerNorm -------------------------------------------------
 * y[r][c] = T(((x[r][c] - mean_r) * rsqrt(var_r + eps) * (1 + scale[s][c]) + shift[s][c]) * post)
 * with mean_r and var_r over the row's cols (fp32, the variance of the
 * differences from the mean) and s = sets[r], or 0 where sets is NULL (n_sets 1).
 * x: x_dtype IMQ_F32 or y_dtype; y_dtype T: bf16 or f16.  shift, scale: fp32
 * [n_sets, cols]; sets: int32 [rows] (clamped to [0, n_sets)): the text and
 * image rows of a joint residual take their own modulation in one launch.
 * post: the 1/16 of the f16 sandwich (dd_ln_mod_prescale), or 1.
 * x and y contiguous [rows, cols], cols up to 2^20; rows 0 is a no-op; y may be x where both
 * have the same type. */
int imq_ln_mod(imq_ctx* ctx, const void* x, imq_dtype x_dtype, const float* shift,
               const float* scale, const int32_t* sets, int n_sets, void* y, imq_dtype y_dtype,
               int rows, int cols, float eps, float post, imq_stream stream);

/* ---- rotary positions, with the per-head RMSNorm before them ---------------
 * For every row r and head h of a group of heads, over the head's x[0..dim):
 *   n[i] = x[i] * rsqrt(mean(x^2) + eps) * weight[i]     (weight NULL: n = x)
 *   the pairs (n[a_j], n[b_j]), j < rot_dim / 2, turned by
 *   angle_j = positions[r][axis(j)] * inv_freq[j] and multiplied by amplitude:
 *     y[a_j] = (n[a_j] cos - n[b_j] sin) * amplitude
 *     y[b_j] = (n[b_j] cos + n[a_j] sin) * amplitude
 *   y[i] = n[i] for i >= rot_dim,
 * all in fp32 (the angle and its reduction in fp64: positions to 2^31), each
 * y rounded to T once.  interleaved 0: a_j = j, b_j = j + rot_dim / 2 (dq_rope);
 * 1: a_j = 2j, b_j = 2j + 1 (dd_rope_interleaved).
 * The pairs are divided among `axes` position axes (1 to 4), sections[a] pairs
 * each (host array, sum rot_dim / 2; NULL: one axis).  positions: int32
 * [rows, axes], inv_freq: fp64 [rot_dim / 2] (radians a position, what scaling
 * for long contexts has made of them included), both device arrays; amplitude:
 * the factor that such a scaling puts on cos and sin, else 1.
 * T: bf16, f16 or f32.  dim even, 2 to 1024; rot_dim even, 0 to dim.
 * One launch for the groups given, 1 or 2: the queries and the keys.  A
 * group's y may be its x with the same strides (in place); otherwise no output
 * overlaps an input or another output.  Head and row strides as they come:
 * columns of a projection's output in, rows of a cache out.  Pointers (the
 * weights' too) and strides of whole 16 bytes, with dim and rot_dim multiples of
 * 16 and dim up to 512, take the vector kernel, anything else a slower one (8192
 * rows of 32 / 8 heads of 80 in bf16: all turned 20 us, 40 of each 124). */
typedef struct imq_rope_heads {
    const void* x;       /* T, element (r, h, i) at r * x_row + h * x_head + i */
    void* y;             /* T, element (r, h, i) at r * y_row + h * y_head + i */
    int heads;
    int64_t x_row, x_head, y_row, y_head;
    const float* weight; /* RMSNorm weight, fp32 [dim], or NULL: no norm */
} imq_rope_heads;

int imq_rope(imq_ctx* ctx, const imq_rope_heads* groups, int n_groups, int rows, int dim,
             int rot_dim, int interleaved, const int32_t* positions, int axes, const int* sections,
             const double* inv_freq, float amplitude, float eps, imq_dtype dtype,
             imq_stream stream);

/* ---- attention -------------------------------------------------------------
 * For every sequence s, query t of its n_q queries and query head h, over the
 * keys j of its n_k keys (key head h / (heads / kv_heads)):
 *   e_j = scale * sum_d q[t][h][d] k[j][h'][d]
 *   e_j = softcap * tanh(e_j / softcap)                  (softcap > 0)
 *   e_j = e_j - slopes[h] * |p - j|,  p = t + n_k - n_q   (slopes not NULL)
 *   key j is seen where causal is 0, or j <= p, or j < prefix_lens[s]
 *   o[t][h][d] = T( sum_j softmax_j(e)_j v[j][h'][d] ) over the keys seen; 0 where none is
 *     (NaN where the seen ones' scores are all -infinity).
 * The last query stands at the last key (p), so a few queries over a cache
 * and a whole prompt are the same call.  Keys that a query does not see do
 * not touch its output, whatever they hold (NaN and infinities included): an
 * output that comes out not finite, with such a value in a key near those that
 * its query sees, is made a second time, by the slower kernel.
 * T: bf16 or f16; scores, softmax and sums in fp32, the softmax's weights
 * rounded to T before the product with v (up to 32 rows in bf16 as two bf16
 * each; by rows, not rounded).
 *
 * A sequence's rows:
 *   q_offsets NULL: its queries are rows 0.. of q + s * q_seq (max_q rows are
 *     there), n_q = q_lens[s], or max_q where q_lens is NULL;
 *   q_offsets [n_seq + 1]: documents packed into one sequence of q_rows rows:
 *     rows q_offsets[s] to q_offsets[s + 1] of q (q_seq is not read, q_lens NULL).
 *   The same for the keys with k_offsets, k_lens, max_k, k_rows, k_seq and v_seq.
 * Output rows follow the queries'; rows that are no query's (behind a
 * sequence's n_q, or behind the last document) are left as they were.
 * max_q and max_k bound n_q and n_k: larger device values are clamped to
 * them, as offsets are to [0, q_rows] and [0, k_rows].
 *
 * dim: 1 to 256.  Up to 128, a multiple of 8, with pointers and strides of
 * whole 16 bytes, the matrix-core kernels run (65 to 127 elements multiplied
 * as 128); anything else takes a kernel of one wave per query and head, 300
 * times slower and more on long prompts (2048 causal rows of 16 / 8 heads in
 * bf16: of 128 elements 42 us, of 136 12.7 ms, of 256 24 ms).  Values are
 * summed with weights of 1 and less, which are divided by their sum at the
 * end: in bf16 those sums have to stay in fp32.  Few queries over many keys
 * split the keys over workgroups: fp32 partial sums go to the workspace that the
 * context keeps per stream (imq_qmm_t's, under the same rules: under stream
 * capture a call that would need a larger one runs unsplit; graphs captured on
 * one stream share its workspace with each other and with calls on it, so that
 * replays of two of them, or one and such a call, are not run at once), and a
 * second kernel joins them in order: results do not depend on timing. */
typedef struct imq_attention_args {
    const void* q;
    const void* k;
    const void* v;
    void* out; /* overlaps no input (out at q, k or v itself is refused) */
    int64_t q_seq, q_row, q_head; /* element strides: sequence, row, head; dims are contiguous */
    int64_t k_seq, k_row, k_head;
    int64_t v_seq, v_row, v_head;
    int64_t out_seq, out_row, out_head;
    int n_seq, heads, kv_heads, dim;
    int max_q, max_k;
    int q_rows, k_rows;           /* rows of packed q (and out), k and v (with the offsets) */
    const int32_t* q_offsets;
    const int32_t* k_offsets;
    const int32_t* q_lens;
    const int32_t* k_lens;
    const int32_t* prefix_lens;   /* [n_seq], or NULL; only with causal */
    const float* slopes;          /* [heads], or NULL; finite, up to 2^20 in size */
    float scale;                  /* finite, > 0; with slopes and no cap from 2^-64 on */
    float softcap;                /* 0: none; else up to 4096: a capped score is right to some
                                     2^-21 of it */
    int causal;
    int dtype;                    /* an imq_dtype */
} imq_attention_args;

int imq_attention(imq_ctx* ctx, const imq_attention_args* args, imq_stream stream);

typedef enum imq_attention_kernel {
    IMQ_ATTENTION_ROWS = 0,  /* one wave per query and head; any sizes, strides and alignment */
    IMQ_ATTENTION_TILES = 1, /* matrix-core tiles of queries, keys staged through LDS */
    IMQ_ATTENTION_FEW = 2    /* up to 32 rows of queries and heads a key head: a wave per key range */
} imq_attention_kernel;

typedef struct imq_attention_plan_info {
    int kernel;             /* an imq_attention_kernel */
    int tile_rows;          /* rows (queries times heads a key head) of a workgroup's tile */
    int splits;             /* key ranges joined by a second kernel (1: keys not split) */
    size_t workspace_bytes; /* fp32 partial sums of a split plan */
} imq_attention_plan_info;

/* The plan of an imq_attention call with its workspace in hand, after the same
 * checks of the arguments, without launching anything. */
int imq_attention_plan(imq_ctx* ctx, const imq_attention_args* args, imq_attention_plan_info* out);

#ifdef __cplusplus
}
#endif
#endif /* IMQ_CORE_H */
