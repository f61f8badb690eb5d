// core_kernels.hpp -- launchers of the kernels behind imq_core.h.  The C entry
// points (core.cpp) check every argument before they call these.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace imq {

hipError_t launch_ln_mod(const void* x, int x_dtype, const float* shift, const float* scale,
                         const int32_t* sets, int n_sets, void* y, int y_dtype, int rows, int cols,
                         float eps, float post, hipStream_t stream);

// One group of heads of a rope launch (imq_rope_heads; strides in elements).
struct RopeGroup {
  const void* x;
  void* y;
  const float* weight;
  int64_t x_row, x_head, y_row, y_head;
  int heads;
};

struct RopeArgs {
  RopeGroup g[2];
  const int32_t* positions;
  const double* inv_freq;
  int groups, rows, dim, rot, axes;
  int section_end[4];  // pairs below section_end[a] belong to axes 0..a
  float amplitude, eps;
};

hipError_t launch_rope(const RopeArgs& a, bool interleaved, int dtype, hipStream_t stream);

// imq_attention_args with the strides in elements, passed to the kernels by value.
struct AttnArgs {
  const void *q, *k, *v;
  void* out;
  int64_t q_seq, q_row, q_head, k_seq, k_row, k_head, v_seq, v_row, v_head;
  int64_t out_seq, out_row, out_head;
  const int32_t *q_offsets, *k_offsets, *q_lens, *k_lens, *prefix_lens;
  const float* slopes;
  int n_seq, heads, kv_heads, dim, max_q, max_k, q_rows, k_rows;
  int causal;
  float scale, softcap;
};

// imq_shared_keys with the strides in elements: keys in front of every sequence's own.
struct AttnShared {
  const void *k, *v;
  int64_t k_row, k_head, v_row, v_head;
  int rows;
};

constexpr int kAttnKeys = 64;  // keys of a tile (attn_tiles_kernel)
constexpr int kFewWaves = 4;   // waves of a workgroup (attn_few_kernel) ...
constexpr int kFewKeys = 32;   // ... and keys of a wave's tile

struct AttnPlan {
  int kernel;     // an imq_attention_kernel
  int tile_rows;  // query rows (queries x heads a key head) of a workgroup
  int splits;     // key ranges
  int first;      // ranks of tiles that go from the last rows back (attn_tiles_kernel)
  int near_hs;    // sequences and key heads taken at a time (attn_tiles_kernel)
  int chunk;      // keys of a range, whole key tiles
  size_t bytes;   // workspace of the partial sums (0: not split)
};

// cus: compute units of the device.
AttnPlan attention_plan(const AttnArgs& a, int cus);
// ws: plan.bytes of device memory, NULL where the plan does not split.
hipError_t launch_attention(const AttnArgs& a, const AttnPlan& plan, float* ws, int dtype,
                            hipStream_t stream);

// How a call behind shared keys runs.
struct SharedPlan {
  int kernel;      // an imq_shared_kernel
  AttnPlan tiles;  // IMQ_SHARED_TILES: of the walk over the shared and the own keys,
  int own0;        // the own ones from its key own0 on
  // IMQ_SHARED_STREAM, _PACKED: rows of the batch against the shared keys, in tiles of s_rows, and
  // the ranges of the shared and of each sequence's own keys.
  int s_rows, s_tiles, s_splits, s_chunk, o_splits, o_chunk;
  size_t bytes;    // workspace of the partial sums
};
// workspace: there is one.
SharedPlan attention_shared_plan(const AttnArgs& a, const AttnShared& sh, int cus, bool workspace);
// ws: plan.bytes of device memory.
hipError_t launch_attention_shared_bf16(const AttnArgs& a, const AttnShared& sh, const SharedPlan& p, float* ws,
                                        hipStream_t stream);
hipError_t launch_attention_shared_f16(const AttnArgs& a, const AttnShared& sh, const SharedPlan& p, float* ws,
                                       hipStream_t stream);

}  // namespace imq
