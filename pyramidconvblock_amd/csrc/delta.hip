// The gated delta rule: what lies between its launches, and the choice between chunks and single steps.
#include "delta_common.h"
#include "kernels.h"

namespace pdw {

void delta_launch_f32(const DeltaArgs& p, bool backward, hipStream_t s);
void delta_launch_f16(const DeltaArgs& p, bool backward, hipStream_t s);
void delta_launch_bf16(const DeltaArgs& p, bool backward, hipStream_t s);

static int padded_dk(int dk) { return dk <= 32 ? 32 : dk <= 64 ? 64 : 128; }
static int padded_dv(int dv) { return (dv + 31) / 32 * 32; }
static long long delta_chunks(long long T) { return (T + kDeltaChunk - 1) / kDeltaChunk; }

static DeltaSizes sizes_of(int dk, int dv, int dtype) {
    const int raw = dtype == kF32 ? 3 : dtype == kF16 ? 2 : 1;
    return DeltaSizes(padded_dk(dk), padded_dv(dv), raw, raw < 2 ? 2 : raw);
}

// Steps up to which a call without gradients goes step by step.
constexpr long long kDeltaFewSteps = 16;
bool delta_few_steps(long long T) { return T <= kDeltaFewSteps; }

static size_t whole(size_t n) { return (n + 255) / 256 * 256; }

size_t delta_states_bytes(long long chains, long long T, int dk, int dv, int dtype) {
    const DeltaSizes z = sizes_of(dk, dv, dtype);
    const size_t n = (size_t)(chains * delta_chunks(T));
    return whole(n * z.state * 2) + whole(n * z.u * 2);
}

// The buffers of one call one after another: f(pointer, bytes) of each.
template <typename F>
static void delta_buffers(DeltaArgs& p, const DeltaSizes& z, bool backward, F f) {
    const size_t n = (size_t)(p.chains * p.NC);
    auto take = [&](auto*& ptr, size_t bytes) { ptr = (std::remove_reference_t<decltype(ptr)>)f(whole(bytes)); };
    take(p.wp, n * z.frag_made * 2);
    take(p.dec, n * 2 * kDeltaChunk * 4);
    if (!backward) {
        take(p.kt, n * z.frag_raw * 2);
        take(p.ub, n * z.cols * 4);
    } else {
        take(p.ka, n * z.frag_raw * 2);
        take(p.ds1, n * z.state * 2);
        take(p.du, n * z.cols * 4);
        take(p.c0, n * (size_t)padded_dk(p.dk) * p.dvp * 4);
    }
}

size_t delta_workspace(long long chains, long long T, int dk, int dv, bool backward, bool states, int dtype) {
    if (!backward && !states && delta_few_steps(T)) return 0;
    DeltaArgs p{};
    p.chains = (int)chains, p.NC = delta_chunks(T), p.dk = dk, p.dvp = padded_dv(dv);
    size_t total = 0;
    delta_buffers(p, sizes_of(dk, dv, dtype), backward, [&](size_t bytes) { return total += bytes, (char*)nullptr; });
    return total + (backward || states ? 0 : delta_states_bytes(chains, T, dk, dv, dtype));
}

static bool pieces(const void* base, const DeltaStrides& s, int d, int es) {
    const long long piece = 16 / es > 8 ? 8 : 16 / es;
    return (uintptr_t)base % 16 == 0 && d % 8 == 0 && s.o % piece == 0 && s.t % piece == 0 && s.w % piece == 0 && s.h % piece == 0;
}

int delta_run(const DeltaArgs& in, void* states, bool backward, void* workspace, size_t workspace_bytes, int dtype, hipStream_t s) {
    DeltaArgs p = in;
    p.NC = delta_chunks(p.T), p.dvp = padded_dv(p.dv);
    if (!backward && !states && delta_few_steps(p.T)) return delta_steps_run(p, dtype, s);
    const size_t need = delta_workspace(p.chains, p.T, p.dk, p.dv, backward, states != nullptr, dtype);
    if (need && (!workspace || workspace_bytes < need))
        return set_error("delta: workspace too small (%zu of %zu bytes)", workspace_bytes, need), 1;
    const DeltaSizes z = sizes_of(p.dk, p.dv, dtype);
    char* at = (char*)workspace;
    delta_buffers(p, z, backward, [&](size_t bytes) { return at += bytes, at - bytes; });
    if (!states) states = at;
    p.s0 = (bf16_t*)states;
    p.u = (bf16_t*)((char*)states + whole((size_t)(p.chains * p.NC) * z.state * 2));
    const int es = dtype == kF32 ? 4 : 2;
    p.vec = (pieces(p.q, p.qs, p.dk, es) ? kVecQ : 0) | (pieces(p.k, p.ks, p.dk, es) ? kVecK : 0) | (pieces(p.v, p.vs, p.dv, es) ? kVecV : 0) |
            (pieces(p.gy, p.ys, p.dv, es) ? kVecGy : 0) | (pieces(p.y, p.ys, p.dv, es) ? kVecY : 0) |
            (pieces(p.gq, p.gqs, p.dk, es) && pieces(p.gk, p.gqs, p.dk, es) ? kVecGqk : 0) | (pieces(p.gv, p.gvs, p.dv, es) ? kVecGv : 0);
    if (dtype == kF32) delta_launch_f32(p, backward, s);
    else if (dtype == kF16) delta_launch_f16(p, backward, s);
    else delta_launch_bf16(p, backward, s);
    return check_launch(backward ? "delta_grads_k" : "delta_out_k");
}

}  // namespace pdw
