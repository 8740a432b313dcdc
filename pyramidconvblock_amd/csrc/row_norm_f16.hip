// Row norms and gated residuals (row_norm.h) of f16 tensors.
#include "row_norm.h"

namespace pdw {
int rows_lanes_f16(int C) { return row_lanes<f16_t>(C); }
void rows_launch_f16(const RowArgs& p, unsigned grid, bool backward, hipStream_t s) { rows_dispatch<f16_t>(p, grid, backward, s); }
}  // namespace pdw
