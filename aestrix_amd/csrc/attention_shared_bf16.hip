// attention_shared_bf16.hip -- attention behind shared keys for T = bf16.
#include "attention_shared.hpp"

namespace imq {
hipError_t launch_attention_shared_bf16(const AttnArgs& a, const AttnShared& sh, const SharedPlan& p, float* ws,
                                     hipStream_t stream) {
  return launch_shared_t<kBf16>(a, sh, p, ws, stream);
}
}  // namespace imq
