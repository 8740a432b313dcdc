// The gated delta rule step by step, for single tokens and a few: u = beta (v - a S^T k), S = a S + k u^T, y = scale S^T q.
//
// Bound by memory: the state, 4 dk dv bytes, is read once and written once; what a token adds is a hundredth of it.  A workgroup has 32 columns
// of a chain's state in registers, from the load through all tokens to the store: a row of 128 bytes to 8 lanes (32 where dv is no multiple of
// four), a wavefront 8 rows at a time.  Both products with the old state go through the rows at once, y = scale (a S^T q + (k.q) u), so a
// token takes one sum over the rows, by lane exchanges and LDS, and one barrier.  All of it in fp32.
#pragma once
#include "delta_common.h"

namespace pdw {

constexpr int kStepCols = 32;

template <typename T, int DK, int CV>
__global__ __launch_bounds__(256) void delta_step_k(DeltaArgs p) {
    constexpr int type = sizeof(T) == 4 ? kF32 : __is_same(T, f16_t) ? kF16 : kBF16;
    constexpr int CL = kStepCols / CV, RG = 256 / CL, NR = (DK + RG - 1) / RG;   // lanes of a row, rows at a time, rows of a lane
    __shared__ float red[2][4][CL][2 * CV + 1];
    const int parts = (p.dv + kStepCols - 1) / kStepCols;
    const long long id = p.first + blockIdx.x;
    const int chain = (int)(id / parts);
    const DeltaChain c(p, chain);
    const int cl = threadIdx.x % CL, rg = threadIdx.x / CL, wave = threadIdx.x >> 6;
    const int at = (int)(id - (long long)chain * parts) * kStepCols + cl * CV;
    const bool on = at < p.dv;   // (CV = 4: dv is a multiple of it)
    const long long state = (long long)chain * p.dk * p.dv + at;
    float s[NR][CV];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
        const int row = rg + n * RG;
#pragma unroll
        for (int i = 0; i < CV; ++i) s[n][i] = 0.f;
        if (p.h0 && on && row < p.dk) load_f32<float, CV>(p.h0 + state + (long long)row * p.dv, s[n]);
    }
    const T *q = (const T*)p.q + c.at(p.qs, c.hk), *k = (const T*)p.k + c.at(p.ks, c.hk), *v = (const T*)p.v + c.at(p.vs, c.hv) + at;
    T* y = (T*)p.y + c.at(p.ys, c.hv) + at;
    for (long long i = 0; i < p.T; ++i) {
        const long long t = c.step(p, i);
        if (i >= c.len) {   // (the same for the whole workgroup)
            if (rg == 0 && on)
#pragma unroll
                for (int j = 0; j < CV; ++j) y[t * p.ys.t + j] = from_f32<T>(0.f);
            continue;
        }
        float kr[NR], qr[NR], vr[CV], la, beta, slope;
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            const int row = rg + n * RG;
            kr[n] = row < p.dk ? to_f32(k[t * p.ks.t + row]) : 0.f;
            qr[n] = row < p.dk ? to_f32(q[t * p.qs.t + row]) : 0.f;
        }
#pragma unroll
        for (int j = 0; j < CV; ++j) vr[j] = on ? to_f32(v[t * p.vs.t + j]) : 0.f;
        log_decay(gate_value(p.g, c.at(p.gs, c.hv) + t * p.gs.t, p.gates_f32, type), p.logits, la, slope);
        write_strength(gate_value(p.b, c.at(p.bs, c.hv) + t * p.bs.t, p.gates_f32, type), p.logits, beta, slope);
        const float a = expf(la);
        float sum[2 * CV + 1];
#pragma unroll
        for (int j = 0; j < 2 * CV + 1; ++j) sum[j] = 0.f;
#pragma unroll
        for (int n = 0; n < NR; ++n) {
#pragma unroll
            for (int j = 0; j < CV; ++j) {
                sum[j] = __builtin_fmaf(s[n][j], kr[n], sum[j]);
                sum[CV + j] = __builtin_fmaf(s[n][j], qr[n], sum[CV + j]);
            }
            sum[2 * CV] = __builtin_fmaf(kr[n], qr[n], sum[2 * CV]);
        }
#pragma unroll
        for (int j = 0; j < 2 * CV + 1; ++j) {
            if constexpr (CL <= 8) sum[j] += __shfl_xor(sum[j], 8);
            if constexpr (CL <= 16) sum[j] = swap_add16(sum[j]);
            sum[j] = swap_add32(sum[j]);
        }
        float(&buf)[4][CL][2 * CV + 1] = red[i & 1];
        if ((threadIdx.x & 63) < CL)
#pragma unroll
            for (int j = 0; j < 2 * CV + 1; ++j) buf[wave][cl][j] = sum[j];
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 2 * CV + 1; ++j) sum[j] = (buf[0][cl][j] + buf[1][cl][j]) + (buf[2][cl][j] + buf[3][cl][j]);
        float u[CV], out[CV];
#pragma unroll
        for (int j = 0; j < CV; ++j) {
            u[j] = beta * __builtin_fmaf(-a, sum[j], vr[j]);
            out[j] = p.scale * __builtin_fmaf(a, sum[CV + j], sum[2 * CV] * u[j]);
        }
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int j = 0; j < CV; ++j) s[n][j] = __builtin_fmaf(kr[n], u[j], a * s[n][j]);
        if (rg == 0 && on)
#pragma unroll
            for (int j = 0; j < CV; ++j) y[t * p.ys.t + j] = from_f32<T>(out[j]);
    }
    if (!p.last || !on) return;
#pragma unroll
    for (int n = 0; n < NR; ++n) {
        const int row = rg + n * RG;
        if (row < p.dk) store_f32<float, CV>(p.last + state + (long long)row * p.dv, s[n]);
    }
}

}  // namespace pdw
