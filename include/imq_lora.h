/*
 * imq_lora.h -- low-rank adapters of many requests beside a shared 4-bit
 * projection (imq.h).
 *
 * A batch of requests runs one projection W [n, k] together, each row with its
 * request's adapter i = which[row], or none:
 *
 *   u[row] = scale[i] * A_i x[row]                       A_i [r_i, k]
 *   y[row] = T( deq(W) x[row] + B_i u[row] )             B_i [n, r_i]
 *
 * with one rounding to T at the end: sums are held in fp32, and the second product
 * takes u as two values of T, its upper half and what that leaves (16 bits together
 * in bf16; in f16 22, none below 2^-24).  No counterpart in the reference, which has
 * no adapters.
 *
 * Conventions as in imq.h: an imq_status is returned, nothing throws, calls are
 * asynchronous on the given stream and may be captured into a graph, inputs are
 * never written and nothing is allocated: the caller gives the workspace.
 */
#ifndef IMQ_LORA_H
#define IMQ_LORA_H

#include "imq.h"

#ifdef __cplusplus
extern "C" {
#endif

/* A set of adapters, laid out once.  Ranks are filled up to multiples of 16 with
 * zeros (rows of A, columns of B) and the adapters lie behind each other:
 *   a      T [rows, k]   adapter i in rows first[i] to first[i + 1]
 *   b      T             adapter i [n, first[i + 1] - first[i]] from element first[i] * n on
 *   first  int32 [count + 1], multiples of 16, rising from 0 to rows
 *   scale  fp32 [count], an adapter's, or with rank_scales 1 fp32 [rows], one for each
 *          row of A
 * all in device memory; a and b 16-byte aligned.  max_rank: the largest filled-up
 * rank, 16 to 256.
 * In f16 u has f16's range: a row with a u[r] past it has no finite output, and what
 * u's values lose below 2^-24 is up to 2^-25 |B_i[n, r]| of y[n].  So multiply every
 * column of B by the power of two that brings its largest element to between 1 and 2
 * (less, if smaller elements of the column would lose bits), and divide that rank's
 * scale by it: then u[r] is out of range only where B_i[n, r] u[r] is for some n. */
typedef struct imq_lora {
  const void* a;
  const void* b;
  const int32_t* first;
  const float* scale;
  int count, rows, max_rank;
  int rank_scales; /* 0 or 1 */
} imq_lora;

/* Bytes of the workspace of an imq_qmm_lora call of these sizes (16 or more). */
int imq_qmm_lora_workspace(imq_ctx* ctx, const imq_lora* lora, int k, int n, int m, imq_dtype dtype,
                           size_t* bytes);

/* y[m, n] as above.  which: int32 [m] in device memory; a row whose value is not 0 to
 * count - 1 has no adapter.  T is bf16 or f16 (f32: IMQ_EUNSUPPORTED).  ws: at least
 * imq_qmm_lora_workspace's bytes of device memory, 16-byte aligned, this call's alone
 * until its kernels have run.  Other arguments and alignment as imq_qmm_t.  A row's
 * result does not depend on the rows beside it but for the order of fp32 sums, which
 * the sizes alone decide.  What an adapter holds reaches its rows only: where B_i is infinite or
 * NaN, their outputs of that column are not finite. */
int imq_qmm_lora(imq_ctx* ctx, const uint32_t* w, const void* scales, const void* biases,
                 const void* x, const imq_lora* lora, const int32_t* which, void* y, int k, int n,
                 int m, int group_size, int bits, imq_dtype dtype, void* ws, size_t ws_bytes,
                 imq_stream stream);

typedef enum imq_lora_kernel {
  IMQ_LORA_FEW = 0,      /* up to 32 rows: partial sums of K, u beside them in the same launch, a join */
  IMQ_LORA_SPLIT = 1,    /* u, tiles' partial sums (of all of K: splits 1), a join */
  IMQ_LORA_TILES = 2,    /* u, tiles that add B u to their sums */
  IMQ_LORA_TILES_REG = 3 /* the same on the register-staged tiles */
} imq_lora_kernel;

typedef struct imq_lora_plan_info {
  int kernel;     /* an imq_lora_kernel */
  int tile_rows;  /* of the projection's tiles; 0: not in the plan (IMQ_LORA_FEW, _TILES_REG) */
  int splits;     /* ranges of K */
  int u_rows;     /* 1: u a wave for each row and rank; 0: by tiles of 32 rows */
  int grouped;    /* 1: rows are grouped by adapter first (as they are, of more than 1023 adapters) */
  int join_tiles; /* of a join, 1: by tiles of 32 x 32; 0: a thread an output */
  size_t workspace_bytes;
} imq_lora_plan_info;

/* What imq_qmm_lora would run for these sizes, without launching anything. */
int imq_qmm_lora_plan(imq_ctx* ctx, const imq_lora* lora, int k, int n, int m, imq_dtype dtype,
                      imq_lora_plan_info* out);

#ifdef __cplusplus
}
#endif
#endif /* IMQ_LORA_H */
