// qgemm_lora_bf16.hip -- the tile kernels with adapters (EpLora) for T = bf16, K % 256 == 0, and
// the register-staged one.
#include "lora_device.hpp"
#include "qgemm_tile.hpp"

namespace imq {
template hipError_t tile::launch_reg<kBf16, EpLora<kBf16>>(const uint32_t*, const uint16_t*, const uint16_t*,
                                                      const uint16_t*, const EpLora<kBf16>&, int, int,
                                                      int, hipStream_t);
IMQ_TILE_PLAN(kBf16, false, EpLora<kBf16>);
}  // namespace imq
