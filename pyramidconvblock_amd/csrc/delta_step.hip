// Launches of the gated delta rule's form for single tokens (delta_step.h).
#include "delta_step.h"
#include "kernels.h"

namespace pdw {

template <typename T, int DK>
static int steps_launch(DeltaArgs p, bool wide, hipStream_t s) {
    const long long grid = (long long)p.chains * ((p.dv + kStepCols - 1) / kStepCols);
    launch_parts(grid, 256, [&](long long first, unsigned n) {
        p.first = first;
        if (wide) delta_step_k<T, DK, 4><<<n, 256, 0, s>>>(p);
        else delta_step_k<T, DK, 1><<<n, 256, 0, s>>>(p);
    });
    return check_launch("delta_step_k");
}

template <typename T>
static int steps_dispatch(const DeltaArgs& p, bool wide, hipStream_t s) {
    if (p.dk <= 32) return steps_launch<T, 32>(p, wide, s);
    if (p.dk <= 64) return steps_launch<T, 64>(p, wide, s);
    return steps_launch<T, 128>(p, wide, s);
}

int delta_steps_run(const DeltaArgs& p, int dtype, hipStream_t s) {
    const bool wide = p.dv % 4 == 0 && (uintptr_t)p.h0 % 16 == 0 && (uintptr_t)p.last % 16 == 0;
    if (dtype == kF32) return steps_dispatch<float>(p, wide, s);
    if (dtype == kF16) return steps_dispatch<f16_t>(p, wide, s);
    return steps_dispatch<bf16_t>(p, wide, s);
}

}  // namespace pdw
