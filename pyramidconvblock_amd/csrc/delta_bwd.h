// The gated delta rule, backward (names as in delta_fwd.h; d.. is the gradient of .., P = scale G o Q K^T with j <= i):
//
//   dU = P^T dY + E K dS1          Z = (I + A)^-T dU          dV = beta Z
//   dS0 = e^c_end dS1 + scale Q^T D dY - W^T dU
//   dP = dY U^T (j <= i)           dA = -Z U^T (j < i)
//   dQ = scale (D dY S0^T + (G o dP) K)
//   dK = E U dS1^T - D beta Z S0^T + (scale G o dP)^T Q + (M + M^T) K,   M_ij = beta_i G_ij dA_ij
//   dbeta_i = Z_i.V_i - D_i k_i.(Z S0^T)_i + sum_j dA_ij G_ij k_i.k_j
//   dc_i = sum_j N_ij - sum_j N_ji + scale D_i q_i.(dY S0^T)_i - D_i beta_i k_i.(Z S0^T)_i - x_i,   N = dP o P + dA o A,  x_i = E_i k_i.(U dS1^T)_i
//   dc_end += sum_i x_i + e^c_end <S0, dS1>,          d(log a)_t = sum of dc_i over i >= t within the chunk
//
// W and A's blocks are kept from the forward.  delta_back_prepare_k, a workgroup a chunk: dU without dS1's part, and
// C = scale Q^T D dY - W^T dU of that.  delta_chain.h, from the last chunk to the first: dS0 = e^c_end dS1 + C - W^T (E K dS1), the forward's chain with
// the operands' parts exchanged; it leaves the dS1 of every chunk.  delta_grads_k, a workgroup a chunk and key head: all gradients; value heads that
// share a key head one after another, their dQ and dK summed in registers, in one order.
//
// Measured, us a launch (back_prepare, the chains' three, grads), the sizes of delta_fwd.h:
//   bf16, 32 x 3136 x 4 heads of 32 48, 54, 152;  bf16, 8 x 4096 x 6 of 64 48, 42 + 8 + 36, 152;  bf16, 2 x 4096 x 4 and 8 of 128 49, 49 + 13 + 40, 138;
//   fp16, 2 x 16384 x 6 of 64 with a state's gradient 78, 69 + 14 + 39, 237
// delta_back_prepare_k is bound by memory and vector instructions at 32 channels (34 KB a chunk, 4.5 TB/s; they are issued in 83 % of the time).  delta_grads_k, half the
// backward's time, waits: its eight wavefronts meet at six barriers a round of columns and wait for 47 % of their time, vector instructions are issued in 55 %
// (in fp16 with 64 channels, one workgroup a compute unit, 51 and 33 %); two workgroups a compute unit are what LDS and 128 registers hold.
#pragma once
#include "delta_fwd.h"

namespace pdw {

template <typename T, int NP>
__device__ __forceinline__ Half<NP> half_of(const T (&v)[4]) {
    Half<NP> h;
    if constexpr (sizeof(T) == 2 && NP == 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) h.p[0][i] = v[i];
    } else {
        const f32x4 f = {to_f32(v[0]), to_f32(v[1]), to_f32(v[2]), to_f32(v[3])};
        h = split<NP>(f);
    }
    return h;
}

template <typename T, int DK, int MADE>
constexpr int delta_back_prepare_lds() {
    return 2 * delta_rows_bytes<DeltaPlanes<T>::kRaw, DK>() + Blocks<MADE>::kValues * 2 + (int)sizeof(DeltaGates);
}

template <typename T, int DK, int MADE>
constexpr int delta_back_prepare_waves() {
    return delta_waves_of(delta_back_prepare_lds<T, DK, MADE>());
}

// MADE: planes of what the chain's operands are made of: kChainPlanes where the gradient of a state is wanted.
template <typename T, int DK, int MADE>
__global__ __launch_bounds__(256, (delta_back_prepare_waves<T, DK, MADE>())) void delta_back_prepare_k(DeltaArgs p) {
    constexpr int RAW = DeltaPlanes<T>::kRaw;
    // with 32 channels seven workgroups a compute unit wait for one another's loads better than four with their own under way (49 us for 59 at 32 x 3136 steps,
    // 4 heads; with 128 channels 57 us for 49); nor do three planes leave room for them in the 128 registers of four workgroups (64 channels in bf16: 57 us for 66, with
    // spills, at 8 x 4096 steps of 6 heads)
    constexpr bool AHEAD = DK > 32 && !(MADE == kChainPlanes && delta_back_prepare_waves<T, DK, MADE>() == 4);
    typedef Rows<RAW, kDeltaChunk, DK> L;
    extern __shared__ __align__(16) unsigned char lds[];
    bf16_t *q = (bf16_t*)lds, *k = q + L::kValues, *pb = k + L::kValues;
    DeltaGates& s = *(DeltaGates*)(pb + Blocks<MADE>::kValues);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int chain;
    int m;
    if (!chunk_of(p, p.Hv, chain, m)) return;
    const long long id = (long long)chain * p.NC + m;
    const int first = m * kDeltaChunk;
    const DeltaChain c(p, chain);
    const DeltaSizes z(DK, p.dvp, DeltaPlanes<T>::kMade, MADE);
    // columns of v: dU without dS1's part, and C; DK = 32: two wavefronts share a tile of columns where there are few, each half of C's rows
    const int share = p.dvp <= 32 ? 2 : 1, turns = p.dvp / 16 * share;
    // dY's columns (what is not there is read from the first row and dropped)
    T v[4][4];
    auto fetch = [&](int cw, int lane) {
        const int at = cw / share * 16 + (lane & 15);
        const T* gy = (const T*)p.gy + c.at(p.ys, c.hv) + at;
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = first + 16 * b + 4 * (lane >> 4) + r;
                v[b][r] = gy[i < c.len && at < p.dv ? c.step(p, i) * p.ys.t : -(long long)at];
            }
    };

    {
        const int lane = threadIdx.x & 63, col = lane & 15, g4 = 4 * (lane >> 4);
        Run<sizeof(DeltaGates)> gates;
        Staged<T, RAW, DK> ks, qs;
        gates.load(p.gates + id);
        ks.load((const T*)p.k + c.at(p.ks, c.hk), p.ks.t, p, c, first, 0, p.dk, p.vec & kVecK);
        qs.load((const T*)p.q + c.at(p.qs, c.hk), p.qs.t, p, c, first, 0, p.dk, p.vec & kVecQ);
        if (AHEAD && wave < turns) fetch(wave, lane);
        gates.put(&s), ks.put(k), qs.put(q);
        __syncthreads();
        // P's column of blocks: lane = j, values = i
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            if (t < wave) continue;
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int n = 0; n < DK; n += 32) acc = mma<MADE>(L::natural(q, 16 * t, n, lane), L::natural(k, 16 * wave, n, lane), acc);
            const TileDecay decay(s, 16 * wave + col, 16 * t + g4, false);
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[r] = t != wave || col <= g4 + r ? p.scale * decay.G[r] * acc[r] : 0.f;
            Blocks<MADE>::put(pb, Blocks<MADE>::at(t, wave), split<MADE>(acc), lane);
        }
        __syncthreads();
    }
    for (int cw = wave; cw < turns; cw += 4) {
        // (another lane with every turn, for all that the compiler knows: else it reads all of Q^T ahead of the loop, into registers that there are not)
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));
        const int cv = cw / share, part = cw % share, g4 = 4 * (lane >> 4);
        Half<RAW> dr[4];
        Half<MADE> ds[4];
        f32x4 wt[4];   // -W, lane = channel of k, values = steps
        auto fetch_w = [&](int d) {
#pragma unroll
            for (int b = 0; b < 4; ++b) wt[b] = load_at<f32x4>(p.w + id * z.w + d * 1024 + b * 256, lane * 16);
        };
        if (AHEAD) fetch_w(part);
        else fetch(cw, lane);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const f32x4 D = *reinterpret_cast<const f32x4*>(s.D + 16 * b + g4);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (first + 16 * b + g4 + r >= c.len || 16 * cv + (lane & 15) >= p.dv) v[b][r] = from_f32<T>(0.f);
            f32x4 f;
#pragma unroll
            for (int r = 0; r < 4; ++r) f[r] = p.scale * D[r] * to_f32(v[b][r]);
            dr[b] = half_of<T, RAW>(v[b]), ds[b] = split<MADE>(f);
        }
        if (AHEAD && cw + 4 < turns) fetch(cw + 4, lane);
        Half<MADE> us[4];
        float* du = p.du + id * z.cols + cv * 1024;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int t = b; t < 4; ++t) acc = mma(Blocks<MADE>::get(pb, Blocks<MADE>::at(t, b), lane), dr[t], acc);
            if (part == 0) store_at(du + b * 256, lane * 16, acc);
            us[b] = split<MADE>(acc);
        }
        const Frag<MADE> d0 = join(ds[0], ds[1]), d1 = join(ds[2], ds[3]), u0 = join(us[0], us[1]), u1 = join(us[2], us[3]);
        float* c0 = p.c0 + id * z.c0 + cv * (DK * 16);
        for (int d = part; d < DK / 16; d += share) {
            if (!AHEAD) fetch_w(d);
            const Frag<MADE> w0 = join(split<MADE>(wt[0]), split<MADE>(wt[1])), w1 = join(split<MADE>(wt[2]), split<MADE>(wt[3]));
            if (AHEAD && d + share < DK / 16) fetch_w(d + share);
            f32x4 acc = {0.f, 0.f, 0.f, 0.f}, add = acc;
            acc = mma(join(L::down(q, 0, 16 * d, lane), L::down(q, 16, 16 * d, lane)), d0, acc);
            acc = mma(join(L::down(q, 32, 16 * d, lane), L::down(q, 48, 16 * d, lane)), d1, acc);
            add = mma(w0, u0, add);
            add = mma(w1, u1, add);
            store_at(c0 + d * 256, lane * 16, acc + add);
        }
    }
}

// 4 neighbouring values of a row of d, 0 where there are none: as they come, and what they are.
template <typename T>
struct Four {
    typedef unsigned words_t __attribute__((ext_vector_type(sizeof(T))));
    words_t words;
    bool on;
    __device__ __forceinline__ void load(const T* base, long long row, bool there, int at, int d, bool vec) {
        on = there && at < d;
        const T* from = base + (on ? row + at : 0);
        if (vec) {
            words = *reinterpret_cast<const words_t*>(from);
        } else {
            T one[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) one[j] = on && at + j < d ? from[j] : from_f32<T>(0.f);
            __builtin_memcpy(&words, one, sizeof one);
        }
    }
    __device__ __forceinline__ f32x4 values() const {
        T one[4];
        __builtin_memcpy(one, &words, sizeof one);
        f32x4 v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = on ? to_f32(one[j]) : 0.f;
        return v;
    }
};
// The two tiles of a fragment, summed over planes.
template <int NP>
__device__ __forceinline__ void sum_tiles(const Frag<NP>& f, f32x4& lo, f32x4& hi) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        lo[j] = (float)f.p[NP - 1][j], hi[j] = (float)f.p[NP - 1][4 + j];
#pragma unroll
        for (int p = NP - 2; p >= 0; --p) lo[j] += (float)f.p[p][j], hi[j] += (float)f.p[p][4 + j];
    }
}

// Rows of Q and K; in their wake Z's and dY's columns, A's blocks and the states' and U's columns, and in the place of those later the tiles of
// scale G o dP and beta G o dA; gates; sums.
constexpr int kGradsCols = 32, kGradsThreads = 512;
template <typename T, int DK>
struct GradsLds {
    static constexpr int RAW = DeltaPlanes<T>::kRaw, MADE = DeltaPlanes<T>::kMade;
    // (with fp32's three planes and 128 channels the states find no room, and each wavefront turns its own)
    static constexpr bool kStage = !(sizeof(T) == 4 && DK == 128);
    static constexpr int kRows = 2 * Rows<RAW, kDeltaChunk, DK>::kValues;
    static constexpr int kZ = Rows<MADE, kDeltaChunk, kGradsCols>::kValues, kG = Rows<RAW, kDeltaChunk, kGradsCols>::kValues;
    static constexpr int kBlocks = Blocks<MADE>::kValues, kState = 2 * (DK / 32) * MADE * 512, kU = 2 * 2 * MADE * 512;
    static constexpr int kFirst = kZ + kG + kBlocks + (kStage ? 2 * kState + kU : 0), kRounds = kStage ? 1 : 2;
    static constexpr int kSecond = 2 * (kRounds == 1 ? 2 : 1) * Blocks<MADE>::kValues;
    static constexpr int kSums = 3 * 4 * 64 + 4 * 2 * 64 + 8;
    static constexpr int kBytes = (kRows + (kFirst > kSecond ? kFirst : kSecond)) * 2 + (int)sizeof(DeltaGates) + kSums * 4;
};
template <typename T, int DK>
constexpr int delta_grads_lds() {
    return GradsLds<T, DK>::kBytes;
}

// Wavefronts of a SIMD that registers are to be left for: two workgroups of a CU where their LDS lets them be.
template <typename T, int DK, bool SHARED>
constexpr int delta_grads_waves() {
    return !SHARED && delta_grads_lds<T, DK>() <= 80 * 1024 ? 4 : 2;
}

// A sum over 16 neighbouring lanes, in all of them.
__device__ __forceinline__ float sixteen_sum(float v) {
    v = dpp_add<0xB1>(v), v = dpp_add<0x4E>(v), v = dpp_add<0x141>(v);
    return dpp_add<0x140>(v);
}

// Eight wavefronts: each has a block of 16 steps (`row`) and half of the channels of k (`half`): those parts of dQ and dK.  The ten tiles of dP and dA go
// round the wavefronts (lane = step i, values = steps j); what becomes of them goes to all through LDS, both ways round.  SHARED: value
// heads share key heads.
template <typename T, int DK, bool SHARED>
__global__ __launch_bounds__(kGradsThreads, (delta_grads_waves<T, DK, SHARED>())) void delta_grads_k(DeltaArgs p) {
    typedef GradsLds<T, DK> S;
    // the next round's operands under way meanwhile: with shared heads 154 us for 140 (2 x 4096 steps, 4 and 8 heads of 128, bf16), with 128 channels a backward
    // of 523 us for 515 (4 x 4096, 8 heads, bf16); with 64 in fp16 133 for 138, so not there
    constexpr bool AHEAD = SHARED || DK == 128;
    constexpr int RAW = S::RAW, MADE = S::MADE, NT = kGradsThreads, COLS = kGradsCols, ND = DK / 32, NK = DK / 32;   // ND: tiles of this half
    typedef Rows<RAW, kDeltaChunk, DK> L;
    typedef Rows<MADE, kDeltaChunk, COLS> LZ;
    typedef Rows<RAW, kDeltaChunk, COLS> LG;
    extern __shared__ __align__(16) unsigned char lds[];
    bf16_t *q = (bf16_t*)lds, *k = q + L::kValues, *zl = k + L::kValues, *gl = zl + S::kZ, *blocks = gl + S::kG;
    bf16_t *sl = blocks + S::kBlocks, *dl = sl + S::kState, *ul = dl + S::kState;
    bf16_t* tiles = zl;
    DeltaGates& s = *(DeltaGates*)(zl + (S::kFirst > S::kSecond ? S::kFirst : S::kSecond));
    float *rows_n = (float*)(&s + 1), *cols_n = rows_n + 256, *rows_b = cols_n + 256, *dots = rows_b + 256, *inner = dots + 512;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = wave & 3, half = wave >> 2;
    int kchain;
    int m;
    if (!chunk_of(p, p.Hk, kchain, m)) return;
    const int group = SHARED ? p.Hv / p.Hk : 1;
    const int first = m * kDeltaChunk;
    const int chain0 = SHARED ? kchain / p.Hk * p.Hv + kchain % p.Hk * group : kchain;
    const DeltaSizes z(DK, p.dvp, MADE, MADE);
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};

    const DeltaChain ck(p, chain0);
    Staged<T, RAW, DK, NT> ks, qs;
    ks.load((const T*)p.k + ck.at(p.ks, ck.hk), p.ks.t, p, ck, first, 0, p.dk, p.vec & kVecK);
    qs.load((const T*)p.q + ck.at(p.qs, ck.hk), p.qs.t, p, ck, first, 0, p.dk, p.vec & kVecQ);
    f32x4 gq[ND], gk[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) gq[d] = gk[d] = zero;

    for (int e = 0; e < group; ++e) {
        const int chain = chain0 + e;
        const DeltaChain c(p, chain);
        const long long id = (long long)chain * p.NC + m;
        // (a lane that the compiler takes for another one with every head, and in every part below: else it keeps all addresses of all parts, in
        // scratch memory)
        int lane = threadIdx.x & 63;
        if (SHARED) asm volatile("" : "+v"(lane)::"memory");
        const bf16_t *s0 = p.s0 + id * z.state, *ds1 = p.ds1 + id * z.state, *u = p.u + id * z.u;
        // what a round of columns takes: dY, states, U, dU without dS1's part, and V
        Staged<T, RAW, COLS, NT> gs;
        Run<S::kState * 2, NT> rs, rd;
        Run<S::kU * 2, NT> ru;
        f32x4 x[4];
        Four<T> vs;
        auto fetch_v = [&](int at) {
            const int place = first + 16 * row + (lane & 15);
            vs.load((const T*)p.v + c.at(p.vs, c.hv), c.step(p, place) * p.vs.t, place < c.len, at + 16 * half + 4 * (lane >> 4), p.dv, p.vec & kVecV);
        };
        auto fetch_x = [&](int at) {
            if (wave < 2) {
#pragma unroll
                for (int b = 0; b < 4; ++b) x[b] = load_at<f32x4>(p.du + id * z.cols + (at / 16 + wave) * 1024 + b * 256, lane * 16);
            }
        };
        auto fetch = [&](int at) {
            const int cw = at / 16;
            gs.load((const T*)p.gy + c.at(p.ys, c.hv), p.ys.t, p, c, first, at, p.dv, p.vec & kVecGy);
            if constexpr (S::kStage)
                rs.load(s0 + cw * NK * MADE * 512), rd.load(ds1 + cw * NK * MADE * 512), ru.load(u + cw * 2 * MADE * 512);
        };
        {
            Run<sizeof(DeltaGates), NT> gates;
            Run<Blocks<MADE>::kValues * 2, NT> system;
            gates.load(p.gates + id), system.load(p.blocks + id * z.blocks);
            fetch_v(0), fetch(0), fetch_x(0);
            if (e) __syncthreads();
            if (e == 0) ks.put(k), qs.put(q);
            gates.put(&s), system.put(blocks);
        }
        f32x4 aq[ND], az[ND], au[ND];   // dY S0^T, Z S0^T, U dS1^T: lane = step of `row`, values = channels of k
        f32x4 dp[2], da[2];             // dP and -dA of tiles `wave` and wave + 8
#pragma unroll
        for (int d = 0; d < ND; ++d) aq[d] = az[d] = au[d] = zero;
#pragma unroll
        for (int n = 0; n < 2; ++n) dp[n] = da[n] = zero;
        float zv = 0.f, ss = 0.f;       // Z_i.V_i; <S0, dS1>
        for (int at = 0; at < p.dvp; at += COLS) {
            const int cw = at / 16;
            const bool more = at + COLS < p.dvp;
            if (at) {
                if (!AHEAD) fetch_v(at), fetch(at), fetch_x(at);
                __syncthreads();
            }
            if constexpr (S::kStage) rs.put(sl), rd.put(dl), ru.put(ul);
            gs.put(gl);
            __syncthreads();
            if (AHEAD && more) fetch(at + COLS);
            asm volatile("" : "+v"(lane));
            const bf16x4 unit = unit_half(lane);
            // rows of a tile of steps or channels from what lies as the products left it
            auto turned_rows = [&](const bf16_t* staged, const bf16_t* from, int n, int t) {
                if constexpr (S::kStage) {
                    const bf16_t* a = staged + (t / 2) * MADE * 512 + 4 * (t & 1);
                    return join(read_turned<MADE, 8>(a, 512, lane), read_turned<MADE, 8>(a + n * MADE * 512, 512, lane));
                } else {
                    return load_turned<MADE>(from, cw * n + t / 2, n, t & 1, unit, lane);
                }
            };
            if (wave < 2) {
                // dU = that without dS1's part, and E K dS1; then Z
                f32x4 y[4] = {zero, zero, zero, zero};
#pragma unroll
                for (int d = 0; d < NK; ++d) {
                    const Frag<MADE> xs = S::kStage ? load_frag<MADE>(dl, wave * NK + d, lane) : load_frag<MADE>(ds1, (cw + wave) * NK + d, lane);
                    Frag<RAW> a[4];
#pragma unroll
                    for (int b = 0; b < 4; ++b) a[b] = L::tiles(k, 16 * b, 32 * d, lane);
                    mma_rows(a, xs, y);
                }
#pragma unroll
                for (int b = 0; b < 4; ++b) x[b] += y[b] * *reinterpret_cast<const f32x4*>(s.E + 16 * b + 4 * (lane >> 4));
                solve_back<MADE>(blocks, x, lane);
#pragma unroll
                for (int b = 0; b < 4; ++b) LZ::put_turned(zl, 16 * b, 16 * wave, split<MADE>(x[b]), unit, lane);
            }
            if (AHEAD && more) fetch_x(at + COLS);
            // what Z has no part in
            const Frag<MADE> um = turned_rows(ul, u, 2, row);
            {
                const Frag<RAW> om = LG::tiles(gl, 16 * row, 0, lane);
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    const Frag<MADE> sf = turned_rows(sl, s0, NK, half * ND + d), df = turned_rows(dl, ds1, NK, half * ND + d);
                    aq[d] = mma(sf, om, aq[d]);
                    au[d] = mma(df, um, au[d]);
                    if ((d & 3) == row) {
                        f32x4 a0, a1, b0, b1;
                        sum_tiles(sf, a0, a1), sum_tiles(df, b0, b1);
#pragma unroll
                        for (int j = 0; j < 4; ++j) ss = __builtin_fmaf(a0[j], b0[j], __builtin_fmaf(a1[j], b1[j], ss));
                    }
                }
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const int t = wave + 8 * n, b = t < 1 ? 0 : t < 3 ? 1 : t < 6 ? 2 : 3, a = t - b * (b + 1) / 2;
                    if (t < 10) dp[n] = mma(turned_rows(ul, u, 2, a), LG::tiles(gl, 16 * b, 0, lane), dp[n]);
                }
            }
            __syncthreads();
            asm volatile("" : "+v"(lane));
            {
                const int col = lane & 15, g4 = 4 * (lane >> 4);
                const Frag<MADE> zm = LZ::tiles(zl, 16 * row, 0, lane);
#pragma unroll
                for (int d = 0; d < ND; ++d) az[d] = mma(turned_rows(sl, s0, NK, half * ND + d), zm, az[d]);
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const int t = wave + 8 * n, b = t < 1 ? 0 : t < 3 ? 1 : t < 6 ? 2 : 3, a = t - b * (b + 1) / 2;
                    if (t < 10) da[n] = mma(turned_rows(ul, u, 2, a), LZ::tiles(zl, 16 * b, 0, lane), da[n]);
                }
                const int place = first + 16 * row + col, step = c.step(p, place);
                const bool there = place < c.len;
                f32x4 lo, hi;
                sum_tiles(zm, lo, hi);
                if (half) lo = hi;
                const int here = at + 16 * half + g4;
                const f32x4 v = vs.values();
                if (AHEAD && more) fetch_v(at + COLS);
#pragma unroll
                for (int j = 0; j < 4; ++j) zv = __builtin_fmaf(lo[j], v[j], zv);
                if (p.gv && place < p.T)
                    store_four((T*)p.gv + c.at(p.gvs, c.hv) + step * p.gvs.t, here, p.dv, there ? lo * s.beta[16 * row + col] : zero, p.vec & kVecGv);
            }
        }
        __syncthreads();
        asm volatile("" : "+v"(lane));
        const int col = lane & 15, g = lane >> 4, g4 = 4 * g, me = 16 * row + col;
        const bf16x4 unit = unit_half(lane);
        {
            const float D = s.D[me], E = s.E[me], sD = p.scale * D, Db = -D * s.beta[me];
            float qd = 0.f, kz = 0.f, ku = 0.f;
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                const int dc = 16 * (half * ND + d);
                const f32x4 qv = sum_of(L::half(q, 16 * row, dc, lane)), kv = sum_of(L::half(k, 16 * row, dc, lane));
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    qd = __builtin_fmaf(qv[r], aq[d][r], qd);
                    kz = __builtin_fmaf(kv[r], az[d][r], kz);
                    ku = __builtin_fmaf(kv[r], au[d][r], ku);
                }
                gq[d] += aq[d] * sD, gk[d] += az[d] * Db + au[d] * E;
            }
            qd = group_sum(qd), kz = group_sum(kz), ku = group_sum(ku), zv = group_sum(zv);
            const float dot = g == 0 ? qd : g == 1 ? kz : g == 2 ? ku : zv;
            dots[(g * 2 + half) * 64 + me] = dot;
            ss = group_sum(sixteen_sum(ss));
            if (lane == 0) inner[wave] = ss;
        }
        f32x4 xs[2], ys[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const int t = wave + 8 * n, b = t < 1 ? 0 : t < 3 ? 1 : t < 6 ? 2 : 3, a = t - b * (b + 1) / 2;
            if (t >= 10) continue;
            f32x4 qk = zero, kk = zero;
#pragma unroll
            for (int i = 0; i < DK; i += 32) {
                const Frag<RAW> kt = L::natural(k, 16 * a, i, lane);
                qk = mma(kt, L::natural(q, 16 * b, i, lane), qk);
                kk = mma(kt, L::natural(k, 16 * b, i, lane), kk);
            }
            const TileDecay decay(s, 16 * b + col, 16 * a + g4, true);
            float rn = 0.f, rb = 0.f;
            f32x4 cn;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const bool below = a != b || g4 + r < col, at_all = below || (a == b && g4 + r == col);
                const float A = below ? -decay.G[r] * da[n][r] : 0.f;
                xs[n][r] = at_all ? p.scale * decay.G[r] * dp[n][r] : 0.f;
                ys[n][r] = decay.beta[r] * A;
                cn[r] = (below ? xs[n][r] * qk[r] : 0.f) + ys[n][r] * kk[r];   // (the diagonal of N is in both sums: it cancels)
                rn += cn[r], rb += A * kk[r];
            }
            rn = group_sum(rn), rb = group_sum(rb);
            if (g == 0) rows_n[a * 64 + 16 * b + col] = rn, rows_b[a * 64 + 16 * b + col] = rb;
#pragma unroll
            for (int r = 0; r < 4; ++r) cn[r] = sixteen_sum(cn[r]);
            if (col == 0) *reinterpret_cast<f32x4*>(cols_n + b * 64 + 16 * a + g4) = cn;
        }
        // to all: tiles of x and of y, as they are (lane = i) and turned (lane = j)
#pragma unroll
        for (int round = 0; round < S::kRounds; ++round) {
            if (round) __syncthreads();
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const int t = wave + 8 * n;
                if (t >= 10) continue;
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    if (S::kRounds == 2 && w != round) continue;
                    bf16_t* to = tiles + (S::kRounds == 1 ? w * 2 : 0) * Blocks<MADE>::kValues;
                    Half<MADE> h = split<MADE>(w ? ys[n] : xs[n]);
                    Blocks<MADE>::put(to, t, h, lane);
#pragma unroll
                    for (int i = 0; i < MADE; ++i) h.p[i] = turned(h.p[i], unit);
                    Blocks<MADE>::put(to + Blocks<MADE>::kValues, t, h, lane);
                }
            }
            __syncthreads();
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                if (S::kRounds == 2 && w != round) continue;
                const bf16_t *t1 = tiles + (S::kRounds == 1 ? w * 2 : 0) * Blocks<MADE>::kValues, *t2 = t1 + Blocks<MADE>::kValues;
#pragma unroll
                for (int j = 0; j < 5; ++j) {
                    const bool mine = j <= row;   // a tile of this row of blocks, else one of this column
                    const int t = mine ? j : j - 1;
                    const Half<MADE> h = mine ? Blocks<MADE>::get(t1, Blocks<MADE>::at(row, t), lane) : Blocks<MADE>::get(t2, Blocks<MADE>::at(t, row), lane);
                    const bf16_t* by = w || mine ? k : q;
#pragma unroll
                    for (int d = 0; d < ND; ++d) {
                        const Half<RAW> r = L::down(by, 16 * t, 16 * (half * ND + d), lane);
                        if (w == 0 && mine) gq[d] = mma(r, h, gq[d]);
                        else gk[d] = mma(r, h, gk[d]);
                    }
                }
            }
        }
        if (wave == 0) {
            // the gates' gradients: a lane has a step
            float n = 0.f, b = 0.f, dot[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int mine = lane >> 4;
                if (t <= mine) n += rows_n[t * 64 + lane], b += rows_b[t * 64 + lane];
                if (t >= mine) n -= cols_n[t * 64 + lane];
                dot[t] = dots[t * 128 + lane] + dots[t * 128 + 64 + lane];
            }
            const float D = s.D[lane], x = s.E[lane] * dot[2];
            // sum of dc over i >= lane; x is subtracted from its own dc and added to the end's, so what is left is the x before this step
            const double dc = n + p.scale * D * dot[0] - D * s.beta[lane] * dot[1];
            double sum = __shfl(sums_up_to(__shfl(dc, 63 - lane)), 63 - lane);   // (lanes the other way round, and back)
            sum += sums_up_to(x) - x;
            float in = 0.f;
#pragma unroll
            for (int w = 0; w < 8; ++w) in += inner[w];
            sum += (double)s.D[kDeltaChunk - 1] * in;
            const int i = first + lane;
            if (i < p.T) {
                const bool there = i < c.len;
                const long long to = c.at(p.ggs, c.hv) + c.step(p, i) * p.ggs.t;
                const float gg = there ? (float)sum * s.slope[lane] : 0.f, gb = there ? (dot[3] - D * dot[1] + b) * s.bslope[lane] : 0.f;
                if (p.gates_f32) {
                    if (p.gg) ((float*)p.gg)[to] = gg;
                    if (p.gb) ((float*)p.gb)[to] = gb;
                } else {
                    if (p.gg) ((T*)p.gg)[to] = from_f32<T>(gg);
                    if (p.gb) ((T*)p.gb)[to] = from_f32<T>(gb);
                }
            }
        }
    }
    const int lane = threadIdx.x & 63, g4 = 4 * (lane >> 4);
    const int place = first + 16 * row + (lane & 15), step = ck.step(p, place);
    const bool there = place < ck.len;
    if (place < p.T) {
        T *rq = (T*)p.gq + ck.at(p.gqs, ck.hk) + step * p.gqs.t, *rk = (T*)p.gk + ck.at(p.gqs, ck.hk) + step * p.gqs.t;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            const int at = 16 * (half * ND + d) + g4;
            if (p.gq) store_four(rq, at, p.dk, there ? gq[d] : zero, p.vec & kVecGqk);
            if (p.gk) store_four(rk, at, p.dk, there ? gk[d] : zero, p.vec & kVecGqk);
        }
    }
}

}  // namespace pdw
