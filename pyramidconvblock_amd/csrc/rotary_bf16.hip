// Head norms with rotated positions (rotary.h) of bf16 tensors.
#include "rotary.h"

namespace pdw {
int rotary_lanes_bf16(int d, int P) { return rotary_lanes<bf16_t>(d, P); }
void rotary_launch_bf16(const RotaryArgs& p, unsigned grid, bool backward, hipStream_t s) { rotary_dispatch<bf16_t>(p, grid, backward, s); }
}  // namespace pdw
