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
// Three launches and more again; W and A's blocks are kept from the forward.  delta_back_prepare_k, a workgroup a chunk: dU without dS1's part, and
// C = scale Q^T D dY - W^T dU of that.  delta_chain.h, from the last chunk to the first: dS0 = e^c_end dS1 + C - W^T (E K dS1), the forward's chain with
// the operands' parts exchanged; it leaves the dS1 of every chunk.  delta_grads_k, a workgroup a chunk and key head: all gradients; value heads that
// share a key head one after another, their dQ and dK summed in registers, in one order.
#pragma once
#include "delta_fwd.h"

#ifndef FRESH
#define FRESH int lane = threadIdx.x & 63; asm volatile("" : "+v"(lane)); const int col = lane & 15, g = lane >> 4, g4 = 4 * g, me = 16 * wave + col; const long long place = first + me; const bool there = place < ck.len; const long long step = ck.step(p, place); (void)g; (void)g4; (void)there; (void)step; (void)col
#endif
#ifndef SB
#define SB __builtin_amdgcn_sched_barrier(0)
#endif
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

// MADE: planes of what the chain's operands are made of: kChainPlanes where the gradient of a state is wanted.
template <typename T, int DK, int MADE>
__global__ __launch_bounds__(256, 4) void delta_back_prepare_k(DeltaArgs p) {
    constexpr int RAW = DeltaPlanes<T>::kRaw;
    typedef Rows<RAW, kDeltaChunk, DK> L;
    extern __shared__ __align__(16) unsigned char lds[];
    bf16_t *q = (bf16_t*)lds, *k = q + L::kValues, *pb = k + L::kValues;
    DeltaGates& s = *(DeltaGates*)(pb + Blocks<MADE>::kValues);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int chain;
    long long m;
    if (!chunk_of(p, p.Hv, chain, m)) return;
    const long long id = chain * p.NC + m, first = m * kDeltaChunk;
    const DeltaChain c(p, chain);
    const DeltaSizes z(DK, p.dvp, DeltaPlanes<T>::kMade, MADE);

    {
        const int lane = threadIdx.x & 63, col = lane & 15, g4 = 4 * (lane >> 4);
        Run<sizeof(DeltaGates)> gates;
        Staged<T, RAW, DK> ks, qs;
        gates.load(p.gates + id);
        ks.load((const T*)p.k + c.at(p.ks, c.hk), p.ks.t, p, c, first, 0, p.dk, p.vec & kVecK);
        qs.load((const T*)p.q + c.at(p.qs, c.hk), p.qs.t, p, c, first, 0, p.dk, p.vec & kVecQ);
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
    // columns of v: dU without dS1's part, and C; DK = 32: two wavefronts share a tile of columns where there are few, each half of C's rows
    const int share = p.dvp <= 32 ? 2 : 1;
    for (int cw = wave; cw < p.dvp / 16 * share; cw += 4) {
        // (another lane with every turn, for all that the compiler knows: else it reads all of Q^T ahead of the loop, into registers that there are not)
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));
        const int cv = cw / share, part = cw % share, col = lane & 15, g4 = 4 * (lane >> 4), at = 16 * cv + col;
        const T* gy = (const T*)p.gy + c.at(p.ys, c.hv) + at;
        Half<RAW> dr[4];
        Half<MADE> ds[4];
        T v[4][4];
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const long long i = first + 16 * b + g4 + r;
                const bool on = i < c.len && at < p.dv;
                v[b][r] = gy[on ? c.step(p, i) * p.ys.t : -(long long)at];   // (what is not there is read from the first row and dropped)
                if (!on) v[b][r] = from_f32<T>(0.f);
            }
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const f32x4 D = *reinterpret_cast<const f32x4*>(s.D + 16 * b + g4);
            f32x4 f;
#pragma unroll
            for (int r = 0; r < 4; ++r) f[r] = p.scale * D[r] * to_f32(v[b][r]);
            dr[b] = half_of<T, RAW>(v[b]), ds[b] = split<MADE>(f);
        }
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
            const float* w = p.w + id * z.w + d * 1024;   // -W, lane = channel of k, values = steps
            f32x4 wt[4];
#pragma unroll
            for (int b = 0; b < 4; ++b) wt[b] = load_at<f32x4>(w + b * 256, lane * 16);
            f32x4 acc = {0.f, 0.f, 0.f, 0.f}, add = acc;
            acc = mma(join(L::down(q, 0, 16 * d, lane), L::down(q, 16, 16 * d, lane)), d0, acc);
            acc = mma(join(L::down(q, 32, 16 * d, lane), L::down(q, 48, 16 * d, lane)), d1, acc);
            add = mma(join(split<MADE>(wt[0]), split<MADE>(wt[1])), u0, add);
            add = mma(join(split<MADE>(wt[2]), split<MADE>(wt[3])), u1, add);
            store_at(c0 + d * 256, lane * 16, acc + add);
        }
    }
}

// 4 neighbouring values of a row of d, 0 where there are none.
template <typename T>
__device__ __forceinline__ f32x4 load_four(const T* row, bool there, int at, int d, bool vec) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (!there || at >= d) return v;
    if (vec) {
        const ChanVec<T, 4> r = *reinterpret_cast<const ChanVec<T, 4>*>(row + at);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = to_f32(r.v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (at + j < d) v[j] = to_f32(row[at + j]);
    }
    return v;
}
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

// Columns of v that a workgroup has in LDS at a time: as many as leave room for two workgroups on a compute unit, or for one.
template <typename T, int DK>
constexpr int delta_grads_cols() {
    return DK == 32 || (sizeof(T) == 4 && DK == 128) ? 32 : 64;
}
template <typename T, int DK>
constexpr int delta_grads_lds() {
    typedef DeltaPlanes<T> P;
    constexpr int COLS = delta_grads_cols<T, DK>();
    return 2 * delta_rows_bytes<P::kRaw, DK>() + (Rows<P::kMade, kDeltaChunk, COLS>::kValues + Rows<P::kRaw, kDeltaChunk, COLS>::kValues) * 2 +
           Blocks<P::kMade>::kValues * 2 + (int)sizeof(DeltaGates) + (2 * kDeltaChunk + 4) * 4;
}

// A wavefront has a block of 16 steps: its rows of dQ, dK, dV.  What of dP and dA concerns them are five tiles ("slots"): those of its row, blocks
// t <= wave (lane = i, its own step, values = j), and those of its column, t >= wave (lane = j, its own step, values = i).  SHARED: value heads share
// key heads.
template <typename T, int DK, bool SHARED>
__global__ __launch_bounds__(256, sizeof(T) == 4 || DK == 128 ? 1 : 2) void delta_grads_k(DeltaArgs p) {
    constexpr int RAW = DeltaPlanes<T>::kRaw, MADE = DeltaPlanes<T>::kMade;
    constexpr int ND = DK / 16, COLS = delta_grads_cols<T, DK>();
    typedef Rows<RAW, kDeltaChunk, DK> L;
    typedef Rows<MADE, kDeltaChunk, COLS> LZ;
    typedef Rows<RAW, kDeltaChunk, COLS> LG;
    extern __shared__ __align__(16) unsigned char lds[];
    bf16_t *q = (bf16_t*)lds, *k = q + L::kValues, *zl = k + L::kValues, *gl = zl + LZ::kValues, *blocks = gl + LG::kValues;
    DeltaGates& s = *(DeltaGates*)(blocks + Blocks<MADE>::kValues);
    float* dcs = (float*)(&s + 1);   // [64]; x [64]; a part of <S0, dS1> from each wavefront
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int kchain;
    long long m;
    if (!chunk_of(p, p.Hk, kchain, m)) return;
    const int group = SHARED ? p.Hv / p.Hk : 1;
    const long long first = m * kDeltaChunk;
    const int chain0 = SHARED ? kchain / p.Hk * p.Hv + kchain % p.Hk * group : kchain;
    const DeltaSizes z(DK, p.dvp, MADE, MADE);
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};

    const DeltaChain ck(p, chain0);
    Staged<T, RAW, DK> ks, qs;
    ks.load((const T*)p.k + ck.at(p.ks, ck.hk), p.ks.t, p, ck, first, 0, p.dk, p.vec & kVecK);
    qs.load((const T*)p.q + ck.at(p.qs, ck.hk), p.qs.t, p, ck, first, 0, p.dk, p.vec & kVecQ);
    f32x4 gq[ND], gk[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) gq[d] = gk[d] = zero;

    for (int e = 0; e < group; ++e) {
        const int chain = chain0 + e;
        const DeltaChain c(p, chain);
        const long long id = chain * p.NC + m;
        // (a lane that the compiler takes for another one with every head: else it keeps all addresses of all heads' passes, in scratch memory)
        int lane = threadIdx.x & 63;
        if (SHARED) asm volatile("" : "+v"(lane)::"memory");
        const int col = lane & 15, g = lane >> 4, g4 = 4 * g;
        const bf16x4 unit = unit_half(lane);
        const int me = 16 * wave + col;   // this lane's step
        const long long place = first + me;
        const bool there = place < ck.len;
        const long long step = ck.step(p, place);
        Run<sizeof(DeltaGates)> gates;
        Run<Blocks<MADE>::kValues * 2> system;
        gates.load(p.gates + id), system.load(p.blocks + id * z.blocks);

        f32x4 aq[ND], az[ND], au[ND];   // dY S0^T, Z S0^T, U dS1^T: lane = step, values = channels of k
        f32x4 dp[5], da[5];             // dP and -dA
#pragma unroll
        for (int d = 0; d < ND; ++d) aq[d] = az[d] = au[d] = zero;
#pragma unroll
        for (int j = 0; j < 5; ++j) dp[j] = da[j] = zero;
        float zv = 0.f, ss = 0.f;       // Z_i.V_i; <S0, dS1>
        const bf16_t *s0 = p.s0 + id * z.state, *ds1 = p.ds1 + id * z.state, *u = p.u + id * z.u;
        float beta;
        for (int at = 0; at < p.dvp; at += COLS) {
            const int cv = at / 16 + wave;
            const bool mine = 16 * wave < COLS && cv < p.dvp / 16;
            Staged<T, RAW, COLS> gs;
            gs.load((const T*)p.gy + c.at(p.ys, c.hv), p.ys.t, p, c, first, at, p.dv, p.vec & kVecGy);
            f32x4 x[4];
            Frag<MADE> xs[DK / 32];
            if (mine) {
                const float* du = p.du + id * z.cols + cv * 1024;
#pragma unroll
                for (int b = 0; b < 4; ++b) x[b] = load_at<f32x4>(du + b * 256, lane * 16);
#pragma unroll
                for (int d = 0; d < DK / 32; ++d) xs[d] = load_frag<MADE>(ds1, cv * (DK / 32) + d, lane);
            }
            if (e || at) __syncthreads();
            if (at == 0) {
                if (e == 0) ks.put(k), qs.put(q);
                gates.put(&s), system.put(blocks);
            }
            gs.put(gl);
            __syncthreads();
            beta = s.beta[me];
            if (mine) {
                // dU = that without dS1's part, and E K dS1
                f32x4 y[4] = {zero, zero, zero, zero};
#pragma unroll
                for (int d = 0; d < DK / 32; ++d) {
                    Frag<RAW> a[4];
#pragma unroll
                    for (int b = 0; b < 4; ++b) a[b] = L::tiles(k, 16 * b, 32 * d, lane);
                    mma_rows(a, xs[d], y);
                }
#pragma unroll
                for (int b = 0; b < 4; ++b) x[b] += y[b] * *reinterpret_cast<const f32x4*>(s.E + 16 * b + g4);
                solve_back<MADE>(blocks, x, lane);
#pragma unroll
                for (int b = 0; b < 4; ++b) LZ::put_turned(zl, 16 * b, 16 * wave, split<MADE>(x[b]), unit, lane);
            }
            __syncthreads();
#pragma unroll 1
            for (int n = 0; n < COLS && at + n < p.dvp; n += 32) {
                FRESH;
                const int here = at + n + g4, cw = (at + n) / 16;
                const Frag<RAW> om = LG::tiles(gl, 16 * wave, n, lane);
                const Frag<MADE> zm = LZ::tiles(zl, 16 * wave, n, lane);
                const Frag<MADE> um = load_turned<MADE>(u, cw * 2 + wave / 2, 2, wave & 1, unit, lane);
                {
                    const T* v = (const T*)p.v + c.at(p.vs, c.hv) + step * p.vs.t;
                    T* gv = (T*)p.gv + c.at(p.gvs, c.hv) + step * p.gvs.t;
                    f32x4 lo, hi;
                    sum_tiles(zm, lo, hi);
                    const f32x4 vl = load_four(v, there, here, p.dv, p.vec & kVecV), vh = load_four(v, there, here + 16, p.dv, p.vec & kVecV);
#pragma unroll
                    for (int j = 0; j < 4; ++j) zv = __builtin_fmaf(lo[j], vl[j], __builtin_fmaf(hi[j], vh[j], zv));
                    if (p.gv && place < p.T) {
                        store_four(gv, here, p.dv, there ? lo * beta : zero, p.vec & kVecGv);
                        store_four(gv, here + 16, p.dv, there ? hi * beta : zero, p.vec & kVecGv);
                    }
                }
#pragma unroll
                for (int j = 0; j < 5; ++j) {
                    const bool row = j <= wave;
                    const int t = row ? j : j - 1;
                    if (row) {
                        const Frag<MADE> uf = load_turned<MADE>(u, cw * 2 + t / 2, 2, t & 1, unit, lane);
                        dp[j] = mma(uf, om, dp[j]);
                        da[j] = mma(uf, zm, da[j]);
                    } else {
                        dp[j] = mma(LG::tiles(gl, 16 * t, n, lane), um, dp[j]);
                        da[j] = mma(LZ::tiles(zl, 16 * t, n, lane), um, da[j]);
                    }
                    SB;
                }
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    const Frag<MADE> sf = load_turned<MADE>(s0, cw * (DK / 32) + d / 2, DK / 32, d & 1, unit, lane);
                    const Frag<MADE> df = load_turned<MADE>(ds1, cw * (DK / 32) + d / 2, DK / 32, d & 1, unit, lane);
                    aq[d] = mma(sf, om, aq[d]);
                    az[d] = mma(sf, zm, az[d]);
                    au[d] = mma(df, um, au[d]);
                    if ((d & 3) == wave) {
                        f32x4 a0, a1, b0, b1;
                        sum_tiles(sf, a0, a1), sum_tiles(df, b0, b1);
#pragma unroll
                        for (int j = 0; j < 4; ++j) ss = __builtin_fmaf(a0[j], b0[j], __builtin_fmaf(a1[j], b1[j], ss));
                    }
                    SB;
                }
            }
        }

        {
        FRESH;
        const float D = s.D[me], E = s.E[me], sD = p.scale * D, Db = -D * beta;
        float qd = 0.f, kz = 0.f, ku = 0.f;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            const f32x4 qv = sum_of(L::half(q, 16 * wave, 16 * d, lane)), kv = sum_of(L::half(k, 16 * wave, 16 * d, lane));
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                qd = __builtin_fmaf(qv[r], aq[d][r], qd);
                kz = __builtin_fmaf(kv[r], az[d][r], kz);
                ku = __builtin_fmaf(kv[r], au[d][r], ku);
            }
            gq[d] += aq[d] * sD, gk[d] += az[d] * Db + au[d] * E;
        }
        float rown = 0.f, coln = 0.f, db = 0.f;
#pragma unroll
        for (int j = 0; j < 5; ++j) {
            const bool row = j <= wave;
            const int t = row ? j : j - 1;
            FRESH;
            // lane = i, values = j: K of the tile by Q of this block; the other way: Q by K
            const bf16_t *far = row ? k : q, *near = row ? q : k;
            f32x4 qk = zero, kk = zero;
#pragma unroll
            for (int n = 0; n < DK; n += 32) {
                qk = mma(L::natural(far, 16 * t, n, lane), L::natural(near, 16 * wave, n, lane), qk);
                kk = mma(L::natural(k, 16 * t, n, lane), L::natural(k, 16 * wave, n, lane), kk);
            }
            const TileDecay decay(s, me, 16 * t + g4, row);
            f32x4 x, y;
            float n = 0.f;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const bool diagonal = t == wave, below = !diagonal || (row ? g4 + r < col : col < g4 + r), at_all = below || (diagonal && g4 + r == col);
                const float A = below ? -decay.G[r] * da[j][r] : 0.f;
                x[r] = at_all ? p.scale * decay.G[r] * dp[j][r] : 0.f;
                y[r] = decay.beta[r] * A;
                n += (below ? x[r] * qk[r] : 0.f) + y[r] * kk[r];   // (the diagonal of N is in both sums: it cancels)
                db += row ? A * kk[r] : 0.f;
            }
            rown += row ? n : 0.f, coln += row ? 0.f : n;
            const Half<MADE> xs = split<MADE>(x), ys = split<MADE>(y);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                const Half<RAW> kt = L::down(k, 16 * t, 16 * d, lane), ft = L::down(far, 16 * t, 16 * d, lane);
                if (row) gq[d] = mma(ft, xs, gq[d]);
                else gk[d] = mma(ft, xs, gk[d]);
                gk[d] = mma(kt, ys, gk[d]);
            }
            SB;
        }
        rown = group_sum(rown), coln = group_sum(coln), db = group_sum(db), zv = group_sum(zv);
        qd = group_sum(qd), kz = group_sum(kz), ku = group_sum(ku) * E;
        if (g == 0) dcs[me] = rown - coln + sD * qd + Db * kz, dcs[kDeltaChunk + me] = ku;
#pragma unroll
        for (int o = 1; o < 64; o *= 2) ss += __shfl_xor(ss, o);
        if (lane == 0) dcs[2 * kDeltaChunk + wave] = ss;
        const float gbeta = (zv - D * kz + db) * s.bslope[me];
        if (p.gb && g == 0 && place < p.T) {
            const long long to = c.at(p.ggs, c.hv) + step * p.ggs.t;
            const float out = there ? gbeta : 0.f;
            if (p.gates_f32) ((float*)p.gb)[to] = out;
            else ((T*)p.gb)[to] = from_f32<T>(out);
        }
        __syncthreads();
        if (wave == 0) {
            // sum of dc over i >= lane; x is subtracted from its own dc and added to the end's, so what is left is the x before this step
            const float own = dcs[kDeltaChunk + lane];
            double sum = dcs[lane], xs = own;
#pragma unroll
            for (int o = 1; o < 64; o *= 2) {
                const double behind = __shfl_down(sum, o), before = __shfl_up(xs, o);
                if (lane + o < 64) sum += behind;
                if (lane >= o) xs += before;
            }
            sum += xs - own;
            sum += (double)s.D[kDeltaChunk - 1] * ((dcs[128] + dcs[129]) + (dcs[130] + dcs[131]));
            const long long i = first + lane;
            if (p.gg && i < p.T) {
                const long long to = c.at(p.ggs, c.hv) + c.step(p, i) * p.ggs.t;
                const float out = i < c.len ? (float)sum * s.slope[lane] : 0.f;
                if (p.gates_f32) ((float*)p.gg)[to] = out;
                else ((T*)p.gg)[to] = from_f32<T>(out);
            }
        }
        }
    }
    const int lane = threadIdx.x & 63, g4 = 4 * (lane >> 4);
    const long long place = first + 16 * wave + (lane & 15), step = ck.step(p, place);
    const bool there = place < ck.len;
    if (place < p.T) {
        T *rq = (T*)p.gq + ck.at(p.gqs, ck.hk) + step * p.gqs.t, *rk = (T*)p.gk + ck.at(p.gqs, ck.hk) + step * p.gqs.t;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            if (p.gq) store_four(rq, 16 * d + g4, p.dk, there ? gq[d] : zero, p.vec & kVecGqk);
            if (p.gk) store_four(rk, 16 * d + g4, p.dk, there ? gk[d] : zero, p.vec & kVecGqk);
        }
    }
}

}  // namespace pdw
