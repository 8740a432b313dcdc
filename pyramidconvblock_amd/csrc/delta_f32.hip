// The gated delta rule (delta_fwd.h, delta_bwd.h) on f32 tensors.
#include "delta_launch.h"

namespace pdw {
void delta_launch_f32(const DeltaArgs& p, bool backward, hipStream_t s) { delta_dispatch<float>(p, backward, s); }
}  // namespace pdw
