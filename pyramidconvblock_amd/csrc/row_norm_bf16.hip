// Row norms and gated residuals (row_norm.h) of bf16 tensors.
#include "row_norm.h"

namespace pdw {
int rows_lanes_bf16(int C) { return row_lanes<bf16_t>(C); }
void rows_launch_bf16(const RowArgs& p, unsigned grid, bool backward, hipStream_t s) { rows_dispatch<bf16_t>(p, grid, backward, s); }
}  // namespace pdw
