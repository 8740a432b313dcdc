// The gated delta rule (delta_fwd.h, delta_bwd.h) on f16 tensors.
#include "delta_launch.h"

namespace pdw {
void delta_launch_f16(const DeltaArgs& p, bool backward, hipStream_t s) { delta_dispatch<f16_t>(p, backward, s); }
}  // namespace pdw
