// lora.hpp -- launchers of the kernels behind imq_lora.h.  The C entry point
// (lora.cpp) checks every argument before it calls these.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace imq {

constexpr int kLoraMaxRank = 256;

// The adapters of a call (imq_lora), passed to the kernels by value.
struct LoraArgs {
  const uint16_t* a;
  const uint16_t* b;
  const int32_t* first;
  const float* scale;
  const int32_t* which;
  float* u;  // [m][max_rank]: scale * A x of each row's adapter
  int count, rows, max_rank;
};

// u of every row (lora.hip).
hipError_t launch_lora_shrink(const LoraArgs& l, const void* x, int k, int m, int dtype,
                              hipStream_t stream);
// y = T(x . deq(W)^T + B u) (qgemm.hip).
hipError_t launch_qgemm_lora(const uint32_t* w, const void* scales, const void* biases, const void* x,
                             const LoraArgs& l, void* y, int k, int n, int m, int dtype,
                             hipStream_t stream);

}  // namespace imq
