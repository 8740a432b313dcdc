// Head norms with rotated positions (rotary.h) of f32 tensors.
#include "rotary.h"

namespace pdw {
int rotary_lanes_f32(int d, int P) { return rotary_lanes<float>(d, P); }
void rotary_launch_f32(const RotaryArgs& p, unsigned grid, bool backward, hipStream_t s) { rotary_dispatch<float>(p, grid, backward, s); }
}  // namespace pdw
