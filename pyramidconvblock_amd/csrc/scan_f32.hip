// The gated linear recurrence (scan.h) on f32 tensors.
#include "scan.h"

namespace pdw {
void scan_launch_f32(const ScanArgs& p, const ScanShape& shape, ScanPass pass, hipStream_t s) { scan_dispatch<float>(p, shape, pass, s); }
}  // namespace pdw
