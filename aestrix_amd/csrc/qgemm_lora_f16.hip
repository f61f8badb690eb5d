// qgemm_lora_f16.hip -- the tile kernels with adapters (EpLora) for T = f16, K % 256 == 0, and
// the register-staged one.
#include "lora_device.hpp"
#include "qgemm_tile.hpp"

namespace imq {
template hipError_t tile::launch_reg<kF16, EpLora<kF16>>(const uint32_t*, const uint16_t*, const uint16_t*,
                                                      const uint16_t*, const EpLora<kF16>&, int, int,
                                                      int, hipStream_t);
IMQ_TILE_PLAN(kF16, false, EpLora<kF16>);
}  // namespace imq
