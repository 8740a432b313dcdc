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
// Three launches again.  delta_back_prepare_k, a workgroup a chunk: W, dU without dS1's part, and C = scale Q^T D dY - W^T dU of that.
// delta_back_chain_k, from the last chunk to the first: dS0 = e^c_end dS1 + C - W^T (E K dS1), the forward's chain with the operands' parts
// exchanged; it leaves the dS1 of every chunk and completes dU.  delta_grads_k, a workgroup a chunk and key head: all gradients; value heads that
// share a key head one after another, their dQ and dK summed in registers, in one order.
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

template <int MADE, int DK>
constexpr int delta_wt_values() {
    return DK / 16 * 2 * MADE * 64 * 8;
}
template <typename T, int DK>
constexpr int delta_back_prepare_k_values() {   // K, and later W^T in its place
    typedef DeltaPlanes<T> P;
    return Rows<P::kRaw, kDeltaChunk, DK>::kValues > delta_wt_values<P::kMade, DK>() ? Rows<P::kRaw, kDeltaChunk, DK>::kValues
                                                                                    : delta_wt_values<P::kMade, DK>();
}
template <typename T, int DK>
constexpr int delta_back_prepare_lds() {
    typedef DeltaPlanes<T> P;
    return delta_rows_bytes<P::kRaw, DK>() + delta_back_prepare_k_values<T, DK>() * 2 + 2 * Blocks<P::kMade>::kValues * 2 + 4 * 16 * 20 * 4 +
           (int)sizeof(DeltaGates);
}

template <typename T, int DK>
__global__ __launch_bounds__(256) void delta_back_prepare_k(DeltaArgs p) {
    constexpr int RAW = DeltaPlanes<T>::kRaw, MADE = DeltaPlanes<T>::kMade;
    constexpr int type = sizeof(T) == 4 ? kF32 : __is_same(T, f16_t) ? kF16 : kBF16;
    typedef Rows<RAW, kDeltaChunk, DK> L;
    extern __shared__ __align__(16) unsigned char lds[];
    bf16_t *q = (bf16_t*)lds, *k = q + L::kValues, *wl = k;
    bf16_t *blocks = k + delta_back_prepare_k_values<T, DK>(), *pb = blocks + Blocks<MADE>::kValues;
    float* tiles = (float*)(pb + Blocks<MADE>::kValues);
    DeltaGates& s = *(DeltaGates*)(tiles + 4 * 16 * 20);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g4 = 4 * (lane >> 4);
    const long long id = p.first + blockIdx.x;
    const int chain = (int)(id / p.NC);
    const long long first = (id - chain * p.NC) * kDeltaChunk;
    const DeltaChain c(p, chain);
    const DeltaSizes z(DK, p.dvp, RAW, MADE);

    chunk_gates(s, p, c, first, type);
    stage_rows<T, RAW, DK>(k, (const T*)p.k + c.at(p.ks, c.hk), p.ks.t, p, c, first, 0, p.dk, p.vec & kVecK);
    stage_rows<T, RAW, DK>(q, (const T*)p.q + c.at(p.qs, c.hk), p.qs.t, p, c, first, 0, p.dk, p.vec & kVecQ);
    __syncthreads();
    float* tile = tiles + wave * 16 * 20;
    make_blocks<RAW, MADE, DK, true>(blocks, tile, k, s, wave, lane);
    Blocks<MADE>::put(blocks, Blocks<MADE>::at(wave, wave), split<MADE>(invert_block<true>(tile, lane)), lane);
    // P's column of blocks: lane = j, values = i
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        if (t < wave) continue;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < DK; n += 32) acc = mma(L::natural(q, 16 * t, n, lane), L::natural(k, 16 * wave, n, lane), acc);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = 16 * t + g4 + r, j = 16 * wave + col;
            acc[r] = j <= i ? p.scale * decay_between(s, i, j) * acc[r] : 0.f;
        }
        Blocks<MADE>::put(pb, Blocks<MADE>::at(t, wave), split<MADE>(acc), lane);
    }
    // K as the chain's first operand
#pragma unroll
    for (int n = 0; n < DK / 32; ++n) store_frag(p.ka + id * z.frag_raw, wave * (DK / 32) + n, L::tiles(k, 16 * wave, 32 * n, lane), lane);
    __syncthreads();
    if (threadIdx.x < 64) {
        float* dec = p.dec + id * 2 * kDeltaChunk;
        dec[lane] = s.D[lane], dec[64 + lane] = s.E[lane];
    }
    // -W^T: lane = channel of k, values = steps
    constexpr int NT = DK / 16 < 4 ? 1 : DK / 64;
    Frag<MADE> wt[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int ct = wave + 4 * n;
        if (ct >= DK / 16) continue;
        f32x4 x[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            x[b] = sum_of(L::down(k, 16 * b, 16 * ct, lane));
#pragma unroll
            for (int r = 0; r < 4; ++r) x[b][r] *= s.beta[16 * b + g4 + r] * s.D[16 * b + g4 + r];
        }
        solve_fore<MADE>(blocks, x, lane);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            wt[n][h] = join(split<MADE>(-x[2 * h]), split<MADE>(-x[2 * h + 1]));
            store_frag(p.wp + id * z.frag_made, 2 * ct + h, wt[n][h], lane);
        }
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int ct = wave + 4 * n;
        if (ct >= DK / 16) continue;
        store_frag(wl, 2 * ct, wt[n][0], lane);
        store_frag(wl, 2 * ct + 1, wt[n][1], lane);
    }
    __syncthreads();
    for (int cv = wave; cv < p.dvp / 16; cv += 4) {
        const int at = 16 * cv + col;
        const T* gy = (const T*)p.gy + c.at(p.ys, c.hv) + at;
        Half<RAW> dr[4];
        Half<MADE> ds[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            T v[4];
            f32x4 f;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = 16 * b + g4 + r;
                const long long i = first + row;
                v[r] = i < c.len && at < p.dv ? gy[c.step(p, i) * p.ys.t] : from_f32<T>(0.f);
                f[r] = p.scale * s.D[row] * to_f32(v[r]);
            }
            dr[b] = half_of<T, RAW>(v), ds[b] = split<MADE>(f);
        }
        Half<MADE> us[4];
        float* du = p.du + id * z.cols + cv * 1024;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int t = b; t < 4; ++t) acc = mma(Blocks<MADE>::get(pb, Blocks<MADE>::at(t, b), lane), dr[t], acc);
            *reinterpret_cast<f32x4*>(du + (b * 64 + lane) * 4) = acc;
            us[b] = split<MADE>(acc);
        }
        const Frag<MADE> d0 = join(ds[0], ds[1]), d1 = join(ds[2], ds[3]), u0 = join(us[0], us[1]), u1 = join(us[2], us[3]);
        float* c0 = p.c0 + id * (long long)DK * p.dvp + cv * (DK * 16);
#pragma unroll
        for (int d = 0; d < DK / 16; ++d) {
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
            acc = mma(join(L::down(q, 0, 16 * d, lane), L::down(q, 16, 16 * d, lane)), d0, acc);
            acc = mma(join(L::down(q, 32, 16 * d, lane), L::down(q, 48, 16 * d, lane)), d1, acc);
            acc = mma(load_frag<MADE>(wl, 2 * d, lane), u0, acc);
            acc = mma(load_frag<MADE>(wl, 2 * d + 1, lane), u1, acc);
            *reinterpret_cast<f32x4*>(c0 + (d * 64 + lane) * 4) = acc;
        }
    }
}

template <typename T, int DK>
__global__ __launch_bounds__(256) void delta_back_chain_k(DeltaArgs p) {
    constexpr int RAW = DeltaPlanes<T>::kRaw, MADE = DeltaPlanes<T>::kMade;
    const int lane = threadIdx.x & 63, waves = blockDim.x >> 6, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g4 = 4 * (lane >> 4), colv = p.dvp / 16;
    int chain, part;
    if (!chain_part(p, (colv + waves - 1) / waves, chain, part)) return;
    const int cv = part * waves + wave;
    if (cv >= colv) return;
    const DeltaSizes z(DK, p.dvp, RAW, MADE);
    const bf16x4 unit = unit_half(lane);
    const int at = 16 * cv + (lane & 15);
    const long long state = (long long)chain * p.dk * p.dv;
    f32x4 x[DK / 16];
    load_state<DK>(x, p.glast ? p.glast + state : nullptr, p.dk, p.dv, at, lane);
    for (long long m = p.NC - 1; m >= 0; --m) {
        const long long id = chain * p.NC + m;
        const bf16_t *wt = p.wp + id * z.frag_made, *ka = p.ka + id * z.frag_raw;
        const float *c0 = p.c0 + id * (long long)DK * p.dvp + cv * (DK * 16), *dec = p.dec + id * 2 * kDeltaChunk;
        float* du = p.du + id * z.cols + cv * 1024;
        bf16_t* ds1 = p.ds1 + id * z.state;
        Frag<MADE> xs[DK / 32];
#pragma unroll
        for (int d = 0; d < DK / 32; ++d) {
            const Half<MADE> a = split<MADE>(x[2 * d]), b = split<MADE>(x[2 * d + 1]);
            store_turned(ds1, (long long)DK * p.dvp, p.dvp, 32 * d, 16 * cv, a, unit, lane);
            store_turned(ds1, (long long)DK * p.dvp, p.dvp, 32 * d + 16, 16 * cv, b, unit, lane);
            xs[d] = join(a, b);
        }
        Half<MADE> e[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int d = 0; d < DK / 32; ++d) y = mma(load_frag<RAW>(ka, b * (DK / 32) + d, lane), xs[d], y);
            y *= *reinterpret_cast<const f32x4*>(dec + 64 + 16 * b + g4);
            f32x4* to = reinterpret_cast<f32x4*>(du + (b * 64 + lane) * 4);
            *to = *to + y;
            e[b] = split<MADE>(y);
        }
        const Frag<MADE> e0 = join(e[0], e[1]), e1 = join(e[2], e[3]);
        const float end = dec[63];
#pragma unroll
        for (int d = 0; d < DK / 16; ++d) {
            f32x4 n = x[d] * end + *reinterpret_cast<const f32x4*>(c0 + (d * 64 + lane) * 4);
            n = mma(load_frag<MADE>(wt, 2 * d, lane), e0, n);
            x[d] = mma(load_frag<MADE>(wt, 2 * d + 1, lane), e1, n);
        }
    }
    store_state<DK>(p.gh0 ? p.gh0 + state : nullptr, x, p.dk, p.dv, at, lane);
}

// 8 neighbouring values of a row of d, 0 where there are none.
template <typename T>
__device__ __forceinline__ void load_eight(T (&v)[8], const T* row, bool there, int at, int d, bool vec) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = from_f32<T>(0.f);
    if (!there || at >= d) return;
    if (vec) {
        constexpr int VEC = 16 / sizeof(T);
#pragma unroll
        for (int m = 0; m < 8 / VEC; ++m) {
            const ChanVec<T, VEC> r = *reinterpret_cast<const ChanVec<T, VEC>*>(row + at + m * VEC);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[m * VEC + j] = r.v[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (at + j < d) v[j] = row[at + j];
    }
}
template <int NP>
__device__ __forceinline__ void sum_eight(const Frag<NP>& f, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        v[j] = (float)f.p[NP - 1][j];
#pragma unroll
        for (int p = NP - 2; p >= 0; --p) v[j] += (float)f.p[p][j];
    }
}
// 8 values of a lane's row of planes in memory [plane][..][ld]
template <int NP>
__device__ __forceinline__ Frag<NP> load_planes(const bf16_t* from, long long plane, int ld, int row, int at, int lane) {
    Frag<NP> f;
#pragma unroll
    for (int n = 0; n < NP; ++n)
        f.p[n] = *reinterpret_cast<const bf16x8*>(from + n * plane + (long long)(row + (lane & 15)) * ld + at + 8 * (lane >> 4));
    return f;
}

template <typename T, int DK>
constexpr int delta_grads_lds() {
    typedef DeltaPlanes<T> P;
    return 2 * delta_rows_bytes<P::kRaw, DK>() + Rows<P::kMade, kDeltaChunk, kDeltaCols>::kValues * 2 + Blocks<P::kMade>::kValues * 2 +
           4 * 16 * 20 * 4 + (int)sizeof(DeltaGates) + (kDeltaChunk + 4) * 4;
}

template <typename T, int DK>
__global__ __launch_bounds__(256) void delta_grads_k(DeltaArgs p) {
    constexpr int RAW = DeltaPlanes<T>::kRaw, MADE = DeltaPlanes<T>::kMade;
    constexpr int type = sizeof(T) == 4 ? kF32 : __is_same(T, f16_t) ? kF16 : kBF16;
    constexpr int ND = DK / 16;
    typedef Rows<RAW, kDeltaChunk, DK> L;
    typedef Rows<MADE, kDeltaChunk, kDeltaCols> LZ;
    extern __shared__ __align__(16) unsigned char lds[];
    bf16_t *q = (bf16_t*)lds, *k = q + L::kValues, *zl = k + L::kValues, *blocks = zl + LZ::kValues;
    float* tiles = (float*)(blocks + Blocks<MADE>::kValues);
    DeltaGates& s = *(DeltaGates*)(tiles + 4 * 16 * 20);
    float* dcs = (float*)(&s + 1);   // [64], and a part of dc_end from each wavefront
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4, g4 = 4 * g;
    const long long block = p.first + blockIdx.x;
    const int kchain = (int)(block / p.NC), group = p.Hv / p.Hk;
    const long long m = block - kchain * p.NC, first = m * kDeltaChunk;
    const int chain0 = kchain / p.Hk * p.Hv + kchain % p.Hk * group;
    const DeltaSizes z(DK, p.dvp, RAW, MADE);
    const bf16x4 unit = unit_half(lane);
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    const int me = 16 * wave + col;   // this lane's step where lanes are steps of the wavefront's block

    const DeltaChain ck(p, chain0);
    stage_rows<T, RAW, DK>(k, (const T*)p.k + ck.at(p.ks, ck.hk), p.ks.t, p, ck, first, 0, p.dk, p.vec & kVecK);
    stage_rows<T, RAW, DK>(q, (const T*)p.q + ck.at(p.qs, ck.hk), p.qs.t, p, ck, first, 0, p.dk, p.vec & kVecQ);
    const long long place = first + me;
    const bool there = place < ck.len;
    const long long step = ck.step(p, place);
    f32x4 gq[ND], gk[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) gq[d] = gk[d] = zero;

    for (int e = 0; e < group; ++e) {
        const int chain = chain0 + e;
        const DeltaChain c(p, chain);
        const long long id = chain * p.NC + m;
        if (e) __syncthreads();
        chunk_gates(s, p, c, first, type);
        __syncthreads();
        float* tile = tiles + wave * 16 * 20;
        make_blocks<RAW, MADE, DK, false>(blocks, tile, k, s, wave, lane);
        Blocks<MADE>::put(blocks, Blocks<MADE>::at(wave, wave), split<MADE>(invert_block<false>(tile, lane)), lane);
        __syncthreads();

        f32x4 aq[ND], az[ND], au[ND];            // dY S0^T, Z S0^T, U dS1^T of the wavefront's steps: lane = step, values = channels of k
        f32x4 dp1[4], dp2[4], da1[4], da2[4];    // dP and -dA: 1: lane = i of this block, values = j; 2: lane = j of this block, values = i
#pragma unroll
        for (int d = 0; d < ND; ++d) aq[d] = az[d] = au[d] = zero;
#pragma unroll
        for (int t = 0; t < 4; ++t) dp1[t] = dp2[t] = da1[t] = da2[t] = zero;
        float zv = 0.f, ss = 0.f;                // Z_i.V_i; <S0, dS1>
        const bf16_t *s0 = p.s0 + id * z.state, *ds1 = p.ds1 + id * z.state, *u = p.u + id * z.u;
        const T *gy = (const T*)p.gy + c.at(p.ys, c.hv), *v = (const T*)p.v + c.at(p.vs, c.hv) + step * p.vs.t;
        T* gv = (T*)p.gv + c.at(p.gvs, c.hv) + step * p.gvs.t;
        const float beta = s.beta[me];
        for (int at = 0; at < p.dvp; at += kDeltaCols) {
            if (at) __syncthreads();
            const int cv = at / 16 + wave;
            if (cv < p.dvp / 16) {
                const float* du = p.du + id * z.cols + cv * 1024;
                f32x4 x[4];
#pragma unroll
                for (int b = 0; b < 4; ++b) x[b] = *reinterpret_cast<const f32x4*>(du + (b * 64 + lane) * 4);
                solve_back<MADE>(blocks, x, lane);
#pragma unroll
                for (int b = 0; b < 4; ++b) store_turned(zl, LZ::kPlane, LZ::kStride, 16 * b, 16 * wave, split<MADE>(x[b]), unit, lane);
            }
            __syncthreads();
#pragma unroll
            for (int n = 0; n < kDeltaCols; n += 32) {
                if (at + n >= p.dvp) break;
                const int here = at + n + 8 * g;
                Frag<RAW> of[4];
                Frag<MADE> zf[4], uf[4];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    zf[t] = LZ::natural(zl, 16 * t, n, lane);
                    uf[t] = load_planes<MADE>(u, (long long)kDeltaChunk * p.dvp, p.dvp, 16 * t, at + n, lane);
                    const long long i = first + 16 * t + col;
                    T o[8];
                    load_eight(o, gy + c.step(p, i) * p.ys.t, i < c.len, here, p.dv, p.vec & kVecGy);
                    of[t] = planes_of<T, RAW>(o);
                }
                // (this block's fragments by a uniform choice: an index that the compiler knows)
                Frag<RAW> om = of[0];
                Frag<MADE> zm = zf[0], um = uf[0];
#pragma unroll
                for (int t = 1; t < 4; ++t)
                    if (t == wave) om = of[t], zm = zf[t], um = uf[t];
                {
                    T vv[8];
                    load_eight(vv, v, there, here, p.dv, p.vec & kVecV);
                    float zs[8];
                    sum_eight(zm, zs);
                    float out[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) zv = __builtin_fmaf(zs[j], to_f32(vv[j]), zv), out[j] = there ? beta * zs[j] : 0.f;
                    if (p.gv && place < p.T) {
                        const f32x4 lo = {out[0], out[1], out[2], out[3]}, hi = {out[4], out[5], out[6], out[7]};
                        store_four(gv, here, p.dv, lo, p.vec & kVecGv);
                        store_four(gv, here + 4, p.dv, hi, p.vec & kVecGv);
                    }
                }
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    if (t <= wave) {
                        dp1[t] = mma(uf[t], om, dp1[t]);
                        da1[t] = mma(uf[t], zm, da1[t]);
                    }
                    if (t >= wave) {
                        dp2[t] = mma(of[t], um, dp2[t]);
                        da2[t] = mma(zf[t], um, da2[t]);
                    }
                }
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    const Frag<MADE> sf = load_planes<MADE>(s0, (long long)DK * p.dvp, p.dvp, 16 * d, at + n, lane);
                    const Frag<MADE> df = load_planes<MADE>(ds1, (long long)DK * p.dvp, p.dvp, 16 * d, at + n, lane);
                    aq[d] = mma(sf, om, aq[d]);
                    az[d] = mma(sf, zm, az[d]);
                    au[d] = mma(df, um, au[d]);
                    if ((d & 3) == wave) {
                        float a[8], b[8];
                        sum_eight(sf, a), sum_eight(df, b);
#pragma unroll
                        for (int j = 0; j < 8; ++j) ss = __builtin_fmaf(a[j], b[j], ss);
                    }
                }
            }
        }

        float rown = 0.f, coln = 0.f, db = 0.f;
        Half<MADE> p1[4], p2[4], a1[4], a2[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            if (t <= wave) {
                f32x4 qk = zero, kk = zero;
#pragma unroll
                for (int n = 0; n < DK; n += 32) {
                    const Frag<RAW> kt = L::natural(k, 16 * t, n, lane);
                    qk = mma(kt, L::natural(q, 16 * wave, n, lane), qk);
                    kk = mma(kt, L::natural(k, 16 * wave, n, lane), kk);
                }
                f32x4 x, y;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = me, j = 16 * t + g4 + r;
                    const float G = j <= i ? decay_between(s, i, j) : 0.f, A = j < i ? G : 0.f;
                    x[r] = p.scale * G * dp1[t][r];
                    y[r] = -beta * A * da1[t][r];
                    rown += x[r] * qk[r] + y[r] * kk[r];
                    db -= A * da1[t][r] * kk[r];
                }
                p1[t] = split<MADE>(x), a1[t] = split<MADE>(y);
            }
            if (t >= wave) {
                f32x4 qk = zero, kk = zero;
#pragma unroll
                for (int n = 0; n < DK; n += 32) {
                    const Frag<RAW> kw = L::natural(k, 16 * wave, n, lane);
                    qk = mma(L::natural(q, 16 * t, n, lane), kw, qk);
                    kk = mma(L::natural(k, 16 * t, n, lane), kw, kk);
                }
                f32x4 x, y;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = 16 * t + g4 + r, j = me;
                    const float G = j <= i ? decay_between(s, i, j) : 0.f, A = j < i ? G : 0.f;
                    x[r] = p.scale * G * dp2[t][r];
                    y[r] = -s.beta[i] * A * da2[t][r];
                    coln += x[r] * qk[r] + y[r] * kk[r];
                }
                p2[t] = split<MADE>(x), a2[t] = split<MADE>(y);
            }
        }
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
            f32x4 a = gq[d] + aq[d] * sD, b = gk[d] + az[d] * Db + au[d] * E;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const Half<RAW> kt = L::down(k, 16 * t, 16 * d, lane);
                if (t <= wave) a = mma(kt, p1[t], a), b = mma(kt, a1[t], b);
                if (t >= wave) b = mma(kt, a2[t], b), b = mma(L::down(q, 16 * t, 16 * d, lane), p2[t], b);
            }
            gq[d] = a, gk[d] = b;
        }
        rown = group_sum(rown), coln = group_sum(coln), db = group_sum(db), zv = group_sum(zv);
        qd = group_sum(qd), kz = group_sum(kz), ku = group_sum(ku) * E;
        if (g == 0) dcs[me] = rown - coln + sD * qd + Db * kz - ku;
        float end = (g == 0 ? ku : 0.f) + s.D[kDeltaChunk - 1] * ss;
#pragma unroll
        for (int o = 1; o < 64; o *= 2) end += __shfl_xor(end, o);
        if (lane == 0) dcs[kDeltaChunk + wave] = end;
        const float gbeta = (zv - D * kz + db) * s.bslope[me];
        if (p.gb && g == 0 && place < p.T) {
            const long long to = c.at(p.ggs, c.hv) + step * p.ggs.t;
            const float out = there ? gbeta : 0.f;
            if (p.gates_f32) ((float*)p.gb)[to] = out;
            else ((T*)p.gb)[to] = from_f32<T>(out);
        }
        __syncthreads();
        if (wave == 0) {
            double sum = dcs[lane];
            if (lane == 63) sum += (double)dcs[64] + dcs[65] + dcs[66] + dcs[67];
#pragma unroll
            for (int o = 1; o < 64; o *= 2) {
                const double other = __shfl_down(sum, o);
                if (lane + o < 64) sum += other;
            }
            const long long i = first + lane;
            if (p.gg && i < p.T) {
                const long long to = c.at(p.ggs, c.hv) + c.step(p, i) * p.ggs.t;
                const float out = i < c.len ? (float)sum * s.slope[lane] : 0.f;
                if (p.gates_f32) ((float*)p.gg)[to] = out;
                else ((T*)p.gg)[to] = from_f32<T>(out);
            }
        }
    }
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
