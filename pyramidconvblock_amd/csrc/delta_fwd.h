// The gated delta rule, forward.  For every chain (a batch element's value head) with a state S of dk x dv:
//
//   u_t = beta_t (v_t - a_t S_(t-1)^T k_t),   S_t = a_t S_(t-1) + k_t u_t^T,   y_t = scale S_t^T q_t
//
// in chunks of 64 steps.  With c the sums of log a from the chunk's start, D = e^c, E = e^(c_end - c), G_ij = e^(c_i - c_j) and S0 the state
// before the chunk, its rows u solve a triangular system:
//
//   (I + A) U = beta (V - D K S0),   A_ij = beta_i G_ij k_i.k_j for j < i          U = Ub - W S0,  (I + A) [W Ub] = [beta D K   beta V]
//   S1 = e^c_end S0 + K^T E U                                                      Y = scale (D Q S0 + (G o Q K^T) U),  j <= i
//
// Launches: delta_prepare_k, a workgroup a chunk: A, then W and Ub by substitution (16 x 16 blocks: the diagonal's are inverted row by
// row in fp32, the rest is products; powers of A, the other way to its inverse, cancel where keys repeat).  delta_chain.h, the only part with an
// order: states through the chunks, in one launch, or in three where chains are few.  It leaves the states before the chunks and U.  delta_out_k, a
// workgroup a chunk again: Y.  64 steps a chunk: what lies between the launches (states, W) falls with longer ones, the triangle's work rises.
//
// Measured, us a launch (prepare, the chains' three, out):
//   bf16, 32 sequences of 3136 steps, 4 heads of 32      66, 70 (without segments), 36
//   bf16, 8 of 4096, 6 heads of 64                       54, 56 + 10 + 51, 42
//   bf16, 2 of 4096, 4 key and 8 value heads of 128      37, 61 + 17 + 41, 32
//   fp16, 2 of 16384, 6 heads of 64                      78, 64 + 14 + 43, 44
//   bf16, 1 of 3136, 4 heads of 32, no gradients         11, 7 + 7 + 8, 5
// delta_prepare_k is bound by vector instructions with 32 channels (1049 a wavefront in bf16, issued in 82 % of the SIMDs' time): splitting solutions into planes
// between products, the inverses, decays.  delta_out_k is bound by memory: 26 KB a chunk at 32 channels in bf16, 4.6 TB/s.
#pragma once
#include "delta_chain.h"

namespace pdw {

template <int RAW, int DK>
constexpr int delta_rows_bytes() {
    return Rows<RAW, kDeltaChunk, DK>::kValues * 2;
}
// Columns of v that a workgroup has in LDS at a time.
template <typename T, int DK>
constexpr int delta_prepare_cols() {
    return DK == 32 ? 32 : 64;
}
template <typename T, int DK>
constexpr int delta_prepare_lds() {
    typedef DeltaPlanes<T> P;
    return delta_rows_bytes<P::kRaw, DK>() + delta_rows_bytes<P::kRaw, delta_prepare_cols<T, DK>()>() + Blocks<kChainPlanes>::kValues * 2 +
           (int)sizeof(DeltaGates);
}

// Wavefronts of a SIMD that registers are to be left for, of workgroups of 256: as many as LDS has room for, up to four.
constexpr int delta_waves_of(int lds) {
    const int n = 160 * 1024 / lds;
    return n > 4 ? 4 : n;
}
template <typename T, int DK>
constexpr int delta_prepare_waves() {
    return delta_waves_of(delta_prepare_lds<T, DK>());
}

template <typename T, int DK>
__global__ __launch_bounds__(256, (delta_prepare_waves<T, DK>())) void delta_prepare_k(DeltaArgs p) {
    constexpr int RAW = DeltaPlanes<T>::kRaw, MADE = kChainPlanes;
    constexpr int type = sizeof(T) == 4 ? kF32 : __is_same(T, f16_t) ? kF16 : kBF16;
    constexpr int COLS = delta_prepare_cols<T, DK>();
    // Where LDS lets four workgroups be, their 128 registers do not hold the system's blocks from tile to tile, which the compiler tries: it is told
    // of another lane with every tile (66 us for 72 at 32 x 3136 steps of 4 heads of 32 in bf16, 54 for 70, with spills, at 8 x 4096 of 6 of 64); the registers of
    // three hold them (37 us, 39 without, with 128 channels in bf16).
    constexpr bool KEEP = delta_prepare_waves<T, DK>() < 4;
    typedef Rows<RAW, kDeltaChunk, DK> L;
    typedef Rows<RAW, kDeltaChunk, COLS> LV;
    extern __shared__ __align__(16) unsigned char lds[];
    bf16_t *k = (bf16_t*)lds, *vl = k + L::kValues, *blocks = vl + LV::kValues;
    DeltaGates& s = *(DeltaGates*)(blocks + Blocks<MADE>::kValues);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g4 = 4 * (lane >> 4);
    int chain;
    int m;
    if (!chunk_of(p, p.Hv, chain, m)) return;
    const long long id = (long long)chain * p.NC + m;
    const int first = m * kDeltaChunk;
    const DeltaChain c(p, chain);

    GateMaker gates;
    Staged<T, RAW, DK> ks;
    Staged<T, RAW, COLS> vs;
    if (wave == 0) gates.load(p, c, first, type);
    ks.load((const T*)p.k + c.at(p.ks, c.hk), p.ks.t, p, c, first, 0, p.dk, p.vec & kVecK);
    vs.load((const T*)p.v + c.at(p.vs, c.hv), p.vs.t, p, c, first, 0, p.dv, p.vec & kVecV);
    if (wave == 0) gates.make(s, p.gates + id, p, type);
    ks.put(k), vs.put(vl);
    __syncthreads();
    // A's blocks of the wavefront's row of blocks: lane = row i of it, values = columns j of block t
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        if (t > wave) continue;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < DK; n += 32) acc = mma<MADE>(L::natural(k, 16 * t, n, lane), L::natural(k, 16 * wave, n, lane), acc);
        const TileDecay decay(s, 16 * wave + col, 16 * t + g4, true);
        acc = decay.beta * decay.G * acc;
        if (t == wave) {
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[r] = g4 + r < col ? acc[r] : 0.f;
            acc = invert_rows(acc, lane);
        } else {
            acc = -acc;
        }
        Blocks<MADE>::put(blocks, Blocks<MADE>::at(wave, t), split<MADE>(acc), lane);
    }
    __syncthreads();

    const DeltaSizes z(DK, p.dvp, DeltaPlanes<T>::kMade, MADE);
    if (p.blocks) {   // for the backward's transposed system, of the planes that it takes
        constexpr int NG = DeltaPlanes<T>::kMade;
        const bf16x4 unit = unit_half(lane);
        for (int n = wave; n < 10; n += 4) {
            const Half<MADE> h = Blocks<MADE>::get(blocks, n, lane);
            Half<NG> t;
#pragma unroll
            for (int i = 0; i < NG; ++i) t.p[i] = turned(h.p[i], unit);
            Blocks<NG>::put(p.blocks + id * z.blocks, n, t, lane);
        }
    }
    auto factor = [&](int b, bool w, int lane) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(s.beta + 16 * b + 4 * (lane >> 4));
        return w ? v * *reinterpret_cast<const f32x4*>(s.D + 16 * b + 4 * (lane >> 4)) : v;
    };
    f32x4 beta[4], decay[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) beta[b] = factor(b, false, lane), decay[b] = factor(b, true, lane);
    unsigned bad = 0;   // tiles of columns with solutions that are none (delta_common.h): of W, then of Ub
    // columns of W, and with them the first ones of Ub; then the others of Ub
    for (int at = 0; at < p.dvp; at += COLS) {
        if (at) {
            __syncthreads();
            vs.put(vl);
            __syncthreads();
        }
        if (at + COLS < p.dvp) vs.load((const T*)p.v + c.at(p.vs, c.hv), p.vs.t, p, c, first, at + COLS, p.dv, p.vec & kVecV);
        const int end = (p.dvp - at < COLS ? p.dvp - at : COLS) / 16;
        for (int ct = (at ? DK / 16 : 0) + wave; ct < DK / 16 + end; ct += 4) {
            const bool w = ct < DK / 16;
            const int cv = ct - DK / 16;
            int lane = threadIdx.x & 63;
            if (!KEEP) asm volatile("" : "+v"(lane));
            f32x4 R[4], x[4], f[4];
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                R[b] = w ? sum_of(L::down(k, 16 * b, 16 * ct, lane)) : sum_of(LV::down(vl, 16 * b, 16 * cv, lane));
                f[b] = KEEP ? w ? decay[b] : beta[b] : factor(b, w, lane);
            }
            solve_fore<MADE>(blocks, R, f, x, lane);
            bad |= __any(x[3][0] != x[3][0]) ? 1u << (w ? ct : DK / 16 + at / 16 + cv) : 0;
            float* to = w ? p.w + id * z.w + ct * 1024 : p.ub + id * z.cols + (at / 16 + cv) * 1024;   // (-W: as the products take it)
#pragma unroll
            for (int b = 0; b < 4; ++b) store_at(to + b * 256, lane * 16, w ? -x[b] : x[b]);
        }
    }
    for (; bad; bad &= bad - 1) {
        // (another lane for all that the compiler knows: else it makes this part's addresses ahead of the loop that is always run)
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));
        const int ct = __builtin_ctz(bad), cv = ct - DK / 16, g4 = 4 * (lane >> 4);
        const bool w = ct < DK / 16;
        const int at = 16 * (w ? ct : cv) + (lane & 15);
        const T* from = w ? (const T*)p.k + c.at(p.ks, c.hk) + at : (const T*)p.v + c.at(p.vs, c.hv) + at;
        const long long stride = w ? p.ks.t : p.vs.t;
        f32x4 R[4], x[4], f[4];
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = first + 16 * b + g4 + r;
                R[b][r] = i < c.len && at < (w ? p.dk : p.dv) ? to_f32(from[c.step(p, i) * stride]) : 0.f;
                f[b][r] = s.beta[i - first] * (w ? s.D[i - first] : 1.f);
            }
        solve_fore_until<MADE>(blocks, R, f, x, lane);
        float* to = w ? p.w + id * z.w + ct * 1024 : p.ub + id * z.cols + cv * 1024;
#pragma unroll
        for (int b = 0; b < 4; ++b) store_at(to + b * 256, lane * 16, w ? -x[b] : x[b]);
    }
}

// acc + P U where rows of U are bad: lane = step of P and of the result, its values columns; U's lanes are columns.
template <int NP>
__device__ __forceinline__ f32x4 product_until(const bf16_t* us, int fragment, const Frag<NP> (&p)[2], f32x4 acc, int step, int lane) {
    auto row = [&](int n, int j) { return 32 * n + 16 * (j / 4) + 4 * (lane >> 4) + j % 4; };
    int first = kDeltaChunk;
#pragma unroll
    for (int n = 1; n >= 0; --n) {
        const u32x4 u = load_at<u32x4>(us + (fragment + n) * NP * 512, lane * 16);
#pragma unroll
        for (int j = 7; j >= 0; --j) first = (u[j / 2] >> (j & 1) * 16 & 0x7f80) == 0x7f80 ? row(n, j) : first;
    }
    first = first_of_groups(first);
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        Frag<NP> u = load_frag<NP>(us, fragment + n, lane);
        u32x4 there;
#pragma unroll
        for (int j = 0; j < 8; j += 2) there[j / 2] = (row(n, j) < first ? 0xffffu : 0) | (row(n, j + 1) < first ? 0xffff0000u : 0);
#pragma unroll
        for (int i = 0; i < NP; ++i) u.p[i] = __builtin_bit_cast(bf16x8, __builtin_bit_cast(u32x4, u.p[i]) & there);
        acc = mma(u, p[n], acc);
        asm volatile("" : "+v"(lane));   // (one after the other: few registers)
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (step >= __shfl(first, 4 * (lane >> 4) + r)) acc[r] = __builtin_nanf("");
    return acc;
}

template <typename T, int DK>
constexpr int delta_out_lds() {
    return 2 * delta_rows_bytes<DeltaPlanes<T>::kRaw, DK>() + (int)sizeof(DeltaGates);
}

// Wavefronts of a SIMD that registers are left for: as many as its loop over columns needs by itself.
template <typename T, int DK>
constexpr int delta_out_waves() {
    return sizeof(T) == 2 ? (DK == 32 ? 5 : DK == 64 ? 4 : 3) : (DK == 128 ? 2 : 3);
}

template <typename T, int DK>
__global__ __launch_bounds__(256, (delta_out_waves<T, DK>())) void delta_out_k(DeltaArgs p) {
    constexpr int RAW = DeltaPlanes<T>::kRaw, MADE = DeltaPlanes<T>::kMade;
    typedef Rows<RAW, kDeltaChunk, DK> L;
    extern __shared__ __align__(16) unsigned char lds[];
    DeltaGates& s = *(DeltaGates*)lds;
    bf16_t *k = (bf16_t*)(lds + sizeof(DeltaGates)), *q = k + L::kValues;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g4 = 4 * (lane >> 4);
    int chain;
    int m;
    if (!chunk_of(p, p.Hv, chain, m)) return;
    const long long id = (long long)chain * p.NC + m;
    const int first = m * kDeltaChunk;
    const DeltaChain c(p, chain);

    Run<sizeof(DeltaGates)> gates;
    Staged<T, RAW, DK> ks, qs;
    ks.load((const T*)p.k + c.at(p.ks, c.hk), p.ks.t, p, c, first, 0, p.dk, p.vec & kVecK);
    qs.load((const T*)p.q + c.at(p.qs, c.hk), p.qs.t, p, c, first, 0, p.dk, p.vec & kVecQ);
    gates.load(p.gates + id);
    // states and U of 16 columns, under way a turn ahead (they lie with lane = column of v, values = rows: first operands of the transposed products
    // as they are)
    const DeltaSizes z(DK, p.dvp, MADE, MADE);
    struct Columns {
        Frag<MADE> s[DK / 32], u[2];
    };
    auto fetch = [&](int cv) {
        Columns f;
#pragma unroll
        for (int n = 0; n < DK / 32; ++n) f.s[n] = load_frag<MADE>(p.s0 + id * z.state, cv * (DK / 32) + n, lane);
#pragma unroll
        for (int n = 0; n < 2; ++n) f.u[n] = load_frag<MADE>(p.u + id * z.u, cv * 2 + n, lane);
        return f;
    };
    Columns next = fetch(0);
    ks.put(k), qs.put(q), gates.put(&s);
    __syncthreads();
    // the wavefront's 16 steps i: scale G_ij q_i.k_j, lane = i, values = j; and its rows of Q
    const int i = 16 * wave + col;
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    Half<MADE> pr[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        f32x4 acc = zero;
        if (t <= wave) {
#pragma unroll
            for (int n = 0; n < DK; n += 32) acc = mma(L::natural(k, 16 * t, n, lane), L::natural(q, 16 * wave, n, lane), acc);
            const TileDecay decay(s, i, 16 * t + g4, true);
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[r] = t != wave || g4 + r <= col ? p.scale * decay.G[r] * acc[r] : 0.f;
        }
        pr[t] = split<MADE>(acc);
    }
    const Frag<MADE> pf[2] = {join(pr[0], pr[1]), join(pr[2], pr[3])};
    Frag<RAW> qf[DK / 32];
#pragma unroll
    for (int n = 0; n < DK / 32; ++n) qf[n] = L::tiles(q, 16 * wave, 32 * n, lane);
    const float D = p.scale * s.D[i];
    const int step = first + i;
    const bool there = step < c.len;
    T* row = (T*)p.y + c.at(p.ys, c.hv) + c.step(p, step) * p.ys.t;
    unsigned bad = 0;   // tiles of columns with results that are none (delta_common.h)
    for (int cv = 0; cv < p.dvp / 16; ++cv) {
        const Columns f = next;
        if (cv + 1 < p.dvp / 16) next = fetch(cv + 1);
        f32x4 acc = zero;
#pragma unroll
        for (int n = 0; n < DK / 32; ++n) acc = mma(f.s[n], qf[n], acc);
        acc *= D;
        acc = mma(f.u[0], pf[0], acc);
        if (wave >= 2) acc = mma(f.u[1], pf[1], acc);
        bad |= __any(__builtin_isunordered(acc[0], acc[1]) || __builtin_isunordered(acc[2], acc[3])) ? 1u << cv : 0;
        if (step < p.T) store_four(row, 16 * cv + g4, p.dv, there ? acc : zero, p.vec & kVecY);
    }
    for (; bad; bad &= bad - 1) {
        // (another lane for all that the compiler knows: else it makes this part's addresses ahead of the loop that is always run)
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));
        const int i = 16 * wave + (lane & 15), g4 = 4 * (lane >> 4), step = first + i;
        const int cv = __builtin_ctz(bad);
        T* row = (T*)p.y + c.at(p.ys, c.hv) + c.step(p, step) * p.ys.t;
        f32x4 acc = zero;
#pragma unroll
        for (int n = 0; n < DK / 32; ++n) acc = mma(load_frag<MADE>(p.s0 + id * z.state, cv * (DK / 32) + n, lane), qf[n], acc);
        acc = product_until(p.u + id * z.u, cv * 2, pf, acc * (p.scale * s.D[i]), i, lane);
        if (step < p.T) store_four(row, 16 * cv + g4, p.dv, step < c.len ? acc : zero, p.vec & kVecY);
    }
}

}  // namespace pdw
