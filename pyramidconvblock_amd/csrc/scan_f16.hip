// The gated linear recurrence (scan.h) on f16 tensors.
#include "scan.h"

namespace pdw {
void scan_launch_f16(const ScanArgs& p, const ScanShape& shape, ScanPass pass, hipStream_t s) { scan_dispatch<f16_t>(p, shape, pass, s); }
}  // namespace pdw
