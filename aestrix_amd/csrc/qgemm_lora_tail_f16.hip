// qgemm_lora_tail_f16.hip -- the tile kernels with adapters (EpLora) for T = f16, K % 256 != 0.
#include "lora_device.hpp"
#include "qgemm_tile.hpp"

namespace imq {
IMQ_TILE_PLAN(kF16, true, EpLora<kF16>);
}  // namespace imq
