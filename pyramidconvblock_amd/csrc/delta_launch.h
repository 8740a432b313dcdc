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

inline long long delta_chunk_grid(const DeltaArgs& p, int H) { return ((long long)p.O * p.W * p.NC + 7) / 8 * 8 * H; }

template <typename T, int DK, bool BACK, int CP, bool MAPS, int WAVES>
void delta_chains_of(const DeltaArgs& p, int cols, hipStream_t s) {
    static std::once_flag once;
    const long long grid = ((long long)p.chains * (MAPS ? p.segments - 1 : p.segments) + 7) / 8 * 8 * ((cols + WAVES - 1) / WAVES);
    delta_launch(delta_chain_k<T, DK, BACK, CP, MAPS, WAVES>, delta_chain_lds<T, DK, CP>(), once, grid, 128 * WAVES, p, s);
}
template <typename T, int DK, bool BACK, int CP, bool MAPS>
void delta_chains(const DeltaArgs& p, hipStream_t s) {
    const int cols = p.dvp / 16 + (MAPS ? DK / 16 : 0);
    if constexpr (delta_least_waves<DK>() < 4)
        if (cols < 4) return delta_chains_of<T, DK, BACK, CP, MAPS, 2>(p, cols, s);
    delta_chains_of<T, DK, BACK, CP, MAPS, 4>(p, cols, s);
}

template <typename T, int DK, bool BACK, int CP>
void delta_all_chains(const DeltaArgs& p, hipStream_t s) {
    if (p.segments > 1) {
        std::once_flag none;
        delta_chains<T, DK, BACK, CP, true>(p, s);
        delta_launch(delta_join_k<T, DK, BACK, CP>, 0, none, (long long)p.chains * (p.dvp / 16), DK * 4, p, s);
    }
    delta_chains<T, DK, BACK, CP, false>(p, s);
}

template <typename T, int DK>
void delta_forward(const DeltaArgs& p, hipStream_t s) {
    static std::once_flag once[2];
    const long long chunks = delta_chunk_grid(p, p.Hv);
    delta_launch(delta_prepare_k<T, DK>, delta_prepare_lds<T, DK>(), once[0], chunks, 256, p, s);
    delta_all_chains<T, DK, false, kChainPlanes>(p, s);
    delta_launch(delta_out_k<T, DK>, delta_out_lds<T, DK>(), once[1], chunks, 256, p, s);
}

template <typename T, int DK, int CP>
void delta_backward(const DeltaArgs& p, hipStream_t s) {
    static std::once_flag once[3];
    const long long chunks = delta_chunk_grid(p, p.Hv);
    delta_launch(delta_back_prepare_k<T, DK, CP>, delta_back_prepare_lds<T, DK, CP>(), once[0], chunks, 256, p, s);
    delta_all_chains<T, DK, true, CP>(p, s);
    if (p.Hv > p.Hk) delta_launch(delta_grads_k<T, DK, true>, delta_grads_lds<T, DK>(), once[1], delta_chunk_grid(p, p.Hk), kGradsThreads, p, s);
    else delta_launch(delta_grads_k<T, DK, false>, delta_grads_lds<T, DK>(), once[2], chunks, kGradsThreads, p, s);
}

// The gradient of an initial state is a result in 32 bits; the others of 16-bit tensors are rounded to those, or (of fp32 gates) hold 17 bits (delta_common.h).
template <typename T, int DK>
void delta_pass(const DeltaArgs& p, bool backward, hipStream_t s) {
    if (!backward) return delta_forward<T, DK>(p, s);
    if constexpr (DeltaPlanes<T>::kMade < kChainPlanes)
        if (!p.gh0) return delta_backward<T, DK, DeltaPlanes<T>::kMade>(p, s);
    delta_backward<T, DK, kChainPlanes>(p, s);
}

template <typename T>
void delta_dispatch(const DeltaArgs& p, bool backward, hipStream_t s) {
    static_assert(delta_grads_lds<T, 128>() <= 160 * 1024 && delta_back_prepare_lds<T, 128, kChainPlanes>() <= 160 * 1024 &&
                      delta_out_lds<T, 128>() <= 160 * 1024,
                  "LDS");
    if (p.dk <= 32) delta_pass<T, 32>(p, backward, s);
    else if (p.dk <= 64) delta_pass<T, 64>(p, backward, s);
    else delta_pass<T, 128>(p, backward, s);
}

}  // namespace pdw
