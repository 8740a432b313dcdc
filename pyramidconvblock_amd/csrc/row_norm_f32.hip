// Row norms and gated residuals (row_norm.h) of f32 tensors.
#include "row_norm.h"

namespace pdw {
int rows_lanes_f32(int C) { return row_lanes<float>(C); }
void rows_launch_f32(const RowArgs& p, unsigned grid, bool backward, hipStream_t s) { rows_dispatch<float>(p, grid, backward, s); }
}  // namespace pdw
