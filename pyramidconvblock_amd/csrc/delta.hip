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

// Chunks of a segment, by what the chains' launches then take, counted in steps (a chunk in a workgroup that has its place: 1.6, 2.7 and 3.5 us for 32, 64
// and 128 channels).  A launch takes its segments' steps as often as it has more workgroups than the chip has places for, the one that leaves
// states at least what memory takes for them (200 chunks a step); the maps' launch and the joining one take 3 more, and 0.3 a segment.  Measured both
// ways, us of the forward's chains: 128 chains of 49 chunks of 32 channels 80 without segments, 91 with 4; 12 chains of 256 chunks of 64 133 with 20 segments
// (the choice), 138 with 11, 149 with 16, 155 with 29; 16 of 64 chunks of 128 120 with 8, 125 with 4, 144 with 13; 4 of 49 of 32 25 with 17, 51 with 4.
static long long segment_chunks(long long chains, long long NC, int DK, int dvp) {
    // (workgroups of four wavefronts that carry columns, of 16 each, and four that fetch: one a compute unit; of two and two: two)
    auto rounds = [&](long long segments, int cols) {
        const bool few = DK == 32 && cols < 4;
        const long long n = chains * segments * (few ? (cols + 1) / 2 : (cols + 3) / 4), places = few ? 512 : 256;
        return (double)((n + places - 1) / places);
    };
    auto memory = [&](double steps) {
        const double least = (double)chains * NC / 200;
        return steps < least ? least : steps;
    };
    const int cols = dvp / 16, more = cols + DK / 16;
    long long best = NC;
    double cost = memory(NC * rounds(1, cols));
    for (long long s = 2; s <= NC && s <= 64; ++s) {
        const long long seg = (NC + s - 1) / s, n = (NC + seg - 1) / seg;
        const double c = seg * rounds(n - 1, more) + memory(seg * rounds(n, cols)) + 0.3 * n + 3;
        if (c < cost) cost = c, best = seg;
    }
    return best < 1 ? 1 : best;
}

// What a call's buffers and launches go by.
struct DeltaPlan {
    DeltaSizes z;
    long long NC, seg;
    int segments, dvp;
    DeltaPlan(long long chains, long long T, int dk, int dv, bool backward, bool state_gradient, int dtype)
        : z(padded_dk(dk), padded_dv(dv), dtype == kF32 ? 3 : 2, dtype == kF32 || !backward || state_gradient ? kChainPlanes : 2),
          NC(delta_chunks(T)), seg(segment_chunks(chains, NC, padded_dk(dk), padded_dv(dv))),
          segments(NC ? (int)((NC + seg - 1) / seg) : 1), dvp(padded_dv(dv)) {}
};

// Steps up to which a call without gradients goes step by step: a step takes 1.6 us (1 to 64 streams of 8 heads of 64 channels in bf16: 10.5 us for 8, 16.5
// for 16, 22.5 for 24), a chunk's launches 20.4 whatever its steps; with 128 channels 37, 61 and 84 against 70, for 256 streams 50, 85 and 120 against 96.
constexpr long long kDeltaFewSteps = 16;
bool delta_few_steps(long long T) { return T <= kDeltaFewSteps; }

static size_t whole(size_t n) { return (n + 255) / 256 * 256; }

// What a forward keeps for its backward, and a forward without one has in its workspace (but for A's blocks), one after another: f(bytes) -> the
// address of each.
template <typename F>
static void delta_kept(DeltaArgs& p, const DeltaPlan& d, bool blocks, F f) {
    const size_t n = (size_t)(p.chains * d.NC);
    auto take = [&](auto*& ptr, size_t bytes) { ptr = (std::remove_reference_t<decltype(ptr)>)f(whole(bytes)); };
    take(p.s0, n * d.z.state * 2);
    take(p.u, n * d.z.u * 2);
    take(p.gates, n * sizeof(DeltaGates));
    take(p.w, n * d.z.w * 4);
    if (blocks) take(p.blocks, n * d.z.blocks * 2);
}
// What else a call has between its launches.
template <typename F>
static void delta_buffers(DeltaArgs& p, const DeltaPlan& d, bool backward, F f) {
    const size_t n = (size_t)(p.chains * d.NC), maps = (size_t)p.chains * (d.segments - 1);
    auto take = [&](auto*& ptr, size_t bytes) { ptr = (std::remove_reference_t<decltype(ptr)>)f(whole(bytes)); };
    take(p.maps, maps * d.z.map * 2);
    take(p.shifts, maps * d.z.shift * 4);
    if (!backward) {
        take(p.ub, n * d.z.cols * 4);
    } else {
        take(p.ds1, n * d.z.state * 2);
        take(p.du, n * d.z.cols * 4);
        take(p.c0, n * d.z.c0 * 4);
    }
}

static size_t states_bytes(long long chains, const DeltaPlan& d, bool blocks) {
    DeltaArgs p{};
    p.chains = (int)chains;
    size_t total = 0;
    delta_kept(p, d, blocks, [&](size_t bytes) { return total += bytes, (char*)nullptr; });
    return total;
}

size_t delta_states_bytes(long long chains, long long T, int dk, int dv, int dtype) {
    return states_bytes(chains, DeltaPlan(chains, T, dk, dv, false, false, dtype), true);
}

static size_t workspace_bytes_of(long long chains, const DeltaPlan& d, bool backward, bool states) {
    DeltaArgs p{};
    p.chains = (int)chains;
    size_t total = 0;
    delta_buffers(p, d, backward, [&](size_t bytes) { return total += bytes, (char*)nullptr; });
    return total + (backward || states ? 0 : states_bytes(chains, d, false));
}

// (the most that a backward takes: with the gradient of a state)
size_t delta_workspace(long long chains, long long T, int dk, int dv, bool backward, bool states, int dtype) {
    if (!backward && !states && delta_few_steps(T)) return 0;
    return workspace_bytes_of(chains, DeltaPlan(chains, T, dk, dv, backward, true, dtype), backward, states);
}

__global__ __launch_bounds__(256) void delta_through_k(const float* from, float* to, long long n, long long first) {
    const long long i = (first + blockIdx.x) * 256 + threadIdx.x;
    if (i < n) to[i] = from ? from[i] : 0.f;
}
static int delta_states_through(const float* from, float* to, long long n, hipStream_t s) {
    launch_parts((n + 255) / 256, 256, [&](long long first, unsigned m) { delta_through_k<<<m, 256, 0, s>>>(from, to, n, first); });
    return check_launch("delta_through_k");
}

static bool pieces(const void* base, const DeltaStrides& s, int d, int es) {
    const long long piece = 16 / es > 8 ? 8 : 16 / es;
    return (uintptr_t)base % 16 == 0 && d % 8 == 0 && s.o % piece == 0 && s.t % piece == 0 && s.w % piece == 0 && s.h % piece == 0;
}

int delta_run(const DeltaArgs& in, void* states, bool backward, void* workspace, size_t workspace_bytes, int dtype, hipStream_t s) {
    DeltaArgs p = in;
    if (!backward && !states && delta_few_steps(p.T)) return delta_steps_run(p, dtype, s);
    const DeltaPlan d(p.chains, p.T, p.dk, p.dv, backward, p.gh0 != nullptr, dtype);
    // (workgroups are counted in 32 bits; the buffers of so many chunks would not fit the card)
    if (p.chains * d.NC > 1 << 28) return set_error("delta: more than 2^28 chunks"), 1;
    p.NC = (int)d.NC, p.dvp = d.dvp, p.seg = (int)d.seg, p.segments = d.segments;
    const size_t need = workspace_bytes_of(p.chains, d, backward, states != nullptr);
    if (need && (!workspace || workspace_bytes < need))
        return set_error("delta: workspace too small (%zu of %zu bytes)", workspace_bytes, need), 1;
    if (!p.NC) {   // no steps: the states go through as they are
        const float* from = backward ? p.glast : p.h0;
        float* to = backward ? p.gh0 : p.last;
        return to ? delta_states_through(from, to, (long long)p.chains * p.dk * p.dv, s) : 0;
    }
    char* at = (char*)workspace;
    delta_buffers(p, d, backward, [&](size_t bytes) { return at += bytes, at - bytes; });
    const bool blocks = states != nullptr;
    if (states) at = (char*)states;
    delta_kept(p, d, blocks, [&](size_t bytes) { return at += bytes, at - bytes; });
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
