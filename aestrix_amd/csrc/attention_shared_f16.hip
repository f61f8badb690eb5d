// attention_shared_f16.hip -- attention behind shared keys for T = f16.
#include "attention_shared.hpp"

namespace imq {
hipError_t launch_attention_shared_f16(const AttnArgs& a, const AttnShared& sh, const SharedPlan& p, float* ws,
                                     hipStream_t stream) {
  return launch_shared_t<kF16>(a, sh, p, ws, stream);
}
}  // namespace imq
