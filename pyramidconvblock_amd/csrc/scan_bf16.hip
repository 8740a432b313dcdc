// The gated linear recurrence (scan.h) on bf16 tensors.
#include "scan.h"

namespace pdw {
void scan_launch_bf16(const ScanArgs& p, const ScanShape& shape, ScanPass pass, hipStream_t s) { scan_dispatch<bf16_t>(p, shape, pass, s); }
}  // namespace pdw
