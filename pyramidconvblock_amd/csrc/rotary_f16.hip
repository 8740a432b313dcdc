// Head norms with rotated positions (rotary.h) of f16 tensors.
#include "rotary.h"

namespace pdw {
int rotary_lanes_f16(int d, int P) { return rotary_lanes<f16_t>(d, P); }
void rotary_launch_f16(const RotaryArgs& p, unsigned grid, bool backward, hipStream_t s) { rotary_dispatch<f16_t>(p, grid, backward, s); }
}  // namespace pdw
