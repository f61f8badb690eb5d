// qgemm_lora_tail_bf16.hip -- the tile kernels with adapters (EpLora) for T = bf16, K % 256 != 0.
#include "lora_device.hpp"
#include "qgemm_tile.hpp"

namespace imq {
IMQ_TILE_PLAN(kBf16, true, EpLora<kBf16>);
}  // namespace imq
