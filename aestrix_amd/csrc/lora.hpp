// lora.hpp -- launchers of the kernels behind imq_lora.h.  The C entry point
// (lora.cpp) checks every argument before it calls these.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "ctx.hpp"
#include "imq_lora.h"

namespace imq {

namespace detail {
// Everything but the device pointers of a call's x, y and workspace (lora.cpp).
int check_lora(imq_ctx* ctx, const char* fn, const imq_lora* l, int k, int n, int m, imq_dtype dtype);
}  // namespace detail

constexpr int kLoraMaxRank = 256;

// The adapters of a call (imq_lora), passed to the kernels by value.
struct LoraArgs {
  const uint16_t* a;
  const uint16_t* b;
  const int32_t* first;
  const float* scale;
  const int32_t* which;
  // u = scale * A x of each row's adapter and rank, as operand fragments of the second product:
  // [32 rows][16 ranks][upper halves, what they leave][64 lanes][8], lane r + 32 h row r's
  // ranks 8 h to 8 h + 8.  Ranks past a row's adapter's are not written.
  uint16_t* u;
  int count, rows, max_rank;
  int rank_scales;  // scale is by rows of A, not by adapters
  // Rows grouped by their adapters (launch_lora_order), or NULL: as they are.  `which` is then
  // the places' (in the workspace), and u stands by places too.
  const int32_t* order;
};
inline size_t lora_u_bytes(int m, int max_rank) {
  return (size_t)((m + 31) / 32) * (max_rank / 16) * 2 * 64 * 8 * sizeof(uint16_t);
}

// How the projection of a call runs.
struct LoraPlan {
  int few;        // the few-row kernel's partial sums, with u beside them (qskinny.hip), ...
  int splits;     // ... or the tile kernels': ranges of K, joined by launch_lora_join; 0: the
                  // tile kernels add B u themselves
  int mt, nt, split_steps;  // their tiles (BigPlan)
  bool order;     // grouped rows (launch_lora_order)
  size_t bytes;   // of the partial sums
};
LoraPlan lora_plan(int k, int n, int m, int count, int max_rank, int dtype);

// About what the two joins take, us (lora.hip): a thread an output reads B's rows, 10 TB/s; tiles of
// 32 x 32, 256 at a time, load every adapter that the rows may name, 3 TB/s.  160 rows of N = 2560 with
// 24 adapters of rank 16 in turn 30.8 us a call with the first and 40.2 with the second, 64 rows of N = 6144
// with one of rank 256 44.6 and 32.9.
double lora_join_few_us(int n, int m, int max_rank);
double lora_join_tiles_us(int n, int m, int count, int max_rank);
// Whether u is made a wave a row and rank, and whether the join has a thread an output (lora.hip).
bool lora_by_rows(int count, int max_rank, bool grouped, int k, int m);
bool lora_join_few(int n, int m, int count, int max_rank);

// Groups the rows by their adapters, those without one last, each group in its rows' order:
// order [m] the row at a place, which_at [m] its adapter (lora.hip).
hipError_t launch_lora_order(const LoraArgs& l, int32_t* order, int32_t* which_at, int m, hipStream_t stream);
// u of every row (lora.hip).
hipError_t launch_lora_shrink(const LoraArgs& l, const void* x, int k, int m, int dtype,
                              hipStream_t stream);
// y = T(sum of the ranges + B u) (lora.hip); part: fp32 [splits][m][n].
hipError_t launch_lora_join(const LoraArgs& l, const float* part, int splits, void* y, int n, int m,
                            int dtype, hipStream_t stream);
// The few-row kernel's partial sums, ws fp32 [splits][m][n], and u beside them (qskinny.hip).
hipError_t launch_qskinny_lora(const uint32_t* w, const void* scales, const void* biases, const void* x,
                               float* ws, const LoraArgs& l, int k, int n, int m, int dtype,
                               hipStream_t stream);
// The projection: partial sums to part where the plan has them, else y (qgemm.hip).
hipError_t launch_qgemm_lora(const LoraPlan& p, const uint32_t* w, const void* scales, const void* biases,
                             const void* x, const LoraArgs& l, float* part, void* y, int k, int n, int m,
                             int dtype, hipStream_t stream);

}  // namespace imq
