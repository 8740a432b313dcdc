// The gated delta rule (delta_fwd.h, delta_bwd.h) on bf16 tensors.
#include "delta_launch.h"

namespace pdw {
void delta_launch_bf16(const DeltaArgs& p, bool backward, hipStream_t s) { delta_dispatch<bf16_t>(p, backward, s); }
}  // namespace pdw
