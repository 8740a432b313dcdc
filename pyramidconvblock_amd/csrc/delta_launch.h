// Launches of the gated delta rule's kernels for tensors of one type (one source file for each type compiles them).
#pragma once
#include <mutex>

#include "delta_bwd.h"
#include "kernels.h"

namespace pdw {

template <typename K>
inline void delta_launch(K kernel, int lds, std::once_flag& once, long long grid, int threads, DeltaArgs p, hipStream_t s) {
    if (lds > 64 * 1024) std::call_once(once, [&] { (void)hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024); });
    launch_parts(grid, threads, [&](long long first, unsigned n) {
        p.first = first;
        kernel<<<n, threads, lds, s>>>(p);
    });
}

inline long long delta_chain_grid(const DeltaArgs& p, int& waves) {
    const int cols = p.dvp / 16;
    waves = cols < 4 ? cols : 4;
    return ((long long)p.chains + 7) / 8 * 8 * ((cols + waves - 1) / waves);
}

template <typename T, int DK>
void delta_forward(const DeltaArgs& p, hipStream_t s) {
    static std::once_flag once[2];
    const long long chunks = p.chains * p.NC;
    int waves;
    const long long chains = delta_chain_grid(p, waves);
    if (chunks) delta_launch(delta_prepare_k<T, DK>, delta_prepare_lds<T, DK>(), once[0], chunks, 256, p, s);
    std::once_flag none;
    delta_launch(delta_chain_k<T, DK>, 0, none, chains, 64 * waves, p, s);
    if (chunks) delta_launch(delta_out_k<T, DK>, delta_out_lds<T, DK>(), once[1], chunks, 256, p, s);
}

template <typename T, int DK>
void delta_backward(const DeltaArgs& p, hipStream_t s) {
    static std::once_flag once[2];
    const long long chunks = p.chains * p.NC;
    int waves;
    const long long chains = delta_chain_grid(p, waves);
    if (chunks) delta_launch(delta_back_prepare_k<T, DK>, delta_back_prepare_lds<T, DK>(), once[0], chunks, 256, p, s);
    std::once_flag none;
    delta_launch(delta_back_chain_k<T, DK>, 0, none, chains, 64 * waves, p, s);
    if (chunks) delta_launch(delta_grads_k<T, DK>, delta_grads_lds<T, DK>(), once[1], chunks / p.Hv * p.Hk, 256, p, s);
}

template <typename T>
void delta_dispatch(const DeltaArgs& p, bool backward, hipStream_t s) {
    static_assert(delta_grads_lds<T, 128>() <= 160 * 1024 && delta_back_prepare_lds<T, 128>() <= 160 * 1024 && delta_out_lds<T, 128>() <= 160 * 1024, "LDS");
    if (p.dk <= 32) backward ? delta_backward<T, 32>(p, s) : delta_forward<T, 32>(p, s);
    else if (p.dk <= 64) backward ? delta_backward<T, 64>(p, s) : delta_forward<T, 64>(p, s);
    else backward ? delta_backward<T, 128>(p, s) : delta_forward<T, 128>(p, s);
}

}  // namespace pdw
