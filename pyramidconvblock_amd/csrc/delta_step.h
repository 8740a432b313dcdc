// The gated delta rule step by step, for single tokens and a few: u = beta (v - a S^T k), S = a S + k u^T, y = scale S^T q.
//
// Bound by memory: the state, 4 dk dv bytes, is read once and written once; what a token adds is a hundredth of it.  A workgroup has 32 columns
// of a chain's state in registers, from the load through all tokens to the store: a row of 128 bytes to 8 lanes (32 where dv is no multiple of
// four), a wavefront 8 rows at a time.  Both products with the old state go through the rows at once, y = scale (a S^T q + (k.q) u), so a
// token takes one sum over the rows, by lane exchanges and LDS, and one barrier; the next token's rows are on their way meanwhile, and gates are
// made for 64 tokens at a time, a lane each (3.4 us a token without the two).  All of it in fp32.
// Measured: 256 streams of 9 heads of 128 x 128 in bf16 67 us (302 MB of states: 4.5 TB/s); 64 streams of 8 heads of 64 x 64, four tokens, 13.1 us; one
// stream of 16 heads of 64 x 64, one token, 5.1 us a call.
#pragma once
#include "delta_common.h"

namespace pdw {

constexpr int kStepCols = 32;

template <typename T, int DK, int CV>
__global__ __launch_bounds__(256) void delta_step_k(DeltaArgs p) {
    constexpr int type = sizeof(T) == 4 ? kF32 : __is_same(T, f16_t) ? kF16 : kBF16;
    constexpr int CL = kStepCols / CV, RG = 256 / CL, NR = (DK + RG - 1) / RG;   // lanes of a row, rows at a time, rows of a lane
    constexpr int SUMS = 2 * CV + 1, WIDTH = (SUMS + 3) / 4 * 4;
    __shared__ __align__(16) float red[2][4][CL][WIDTH];
    const int parts = (p.dv + kStepCols - 1) / kStepCols;
    const long long id = p.first + blockIdx.x;
    const int chain = (int)(id / parts);
    const DeltaChain c(p, chain);
    const int cl = threadIdx.x % CL, rg = threadIdx.x / CL, wave = threadIdx.x >> 6;
    const int at = (int)(id - (long long)chain * parts) * kStepCols + cl * CV;
    const bool on = at < p.dv;   // (CV = 4: dv is a multiple of it)
    const long long state = (long long)chain * p.dk * p.dv + at;
    const T *q = (const T*)p.q + c.at(p.qs, c.hk), *k = (const T*)p.k + c.at(p.ks, c.hk), *v = (const T*)p.v + c.at(p.vs, c.hv) + at;
    T* y = (T*)p.y + c.at(p.ys, c.hv) + at;
    struct Token {
        T k[NR], q[NR], v[CV];
    };
    // (what is not there is read from the first row and dropped)
    auto load = [&](int i) {
        Token f;
        const long long t = c.step(p, i);
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            const int row = rg + n * RG, r = row < p.dk ? row : 0;
            f.k[n] = k[t * p.ks.t + r], f.q[n] = q[t * p.qs.t + r];
        }
#pragma unroll
        for (int j = 0; j < CV; ++j) f.v[j] = v[t * p.vs.t + (on ? j : -at)];
        return f;
    };
    Token next;
    if (c.len > 0) next = load(0);
    float s[NR][CV];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
        const int row = rg + n * RG;
#pragma unroll
        for (int i = 0; i < CV; ++i) s[n][i] = 0.f;
        if (p.h0 && on && row < p.dk) load_f32<float, CV>(p.h0 + state + (long long)row * p.dv, s[n]);
    }
    float decays = 0.f, strengths = 0.f;   // of 64 tokens, a lane each
    for (int i = 0; i < c.len; ++i) {
        const Token now = next;
        if (i + 1 < c.len) next = load(i + 1);
        const int lane = threadIdx.x & 63;
        if (!(i & 63) && i + lane < c.len) {
            const long long t = c.step(p, i + lane);
            float la, slope;
            log_decay(gate_value(p.g, c.at(p.gs, c.hv) + t * p.gs.t, p.gates_f32, type), p.logits, la, slope);
            write_strength(gate_value(p.b, c.at(p.bs, c.hv) + t * p.bs.t, p.gates_f32, type), p.logits, strengths, slope);
            decays = expf(la);
        }
        auto of_all = [&](float f) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), i & 63)); };
        const float a = of_all(decays), beta = of_all(strengths);
        float kr[NR], qr[NR], vr[CV];
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            const int row = rg + n * RG;
            kr[n] = row < p.dk ? to_f32(now.k[n]) : 0.f, qr[n] = row < p.dk ? to_f32(now.q[n]) : 0.f;
        }
#pragma unroll
        for (int j = 0; j < CV; ++j) vr[j] = on ? to_f32(now.v[j]) : 0.f;
        float sum[WIDTH];
#pragma unroll
        for (int j = 0; j < WIDTH; ++j) sum[j] = 0.f;
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
        for (int j = 0; j < SUMS; ++j) {
            if constexpr (CL <= 8) sum[j] = dpp_add<0x128>(sum[j]);   // (8 lanes on, round 16)
            if constexpr (CL <= 16) sum[j] = swap_add16(sum[j]);
            sum[j] = swap_add32(sum[j]);
        }
        float(&buf)[4][CL][WIDTH] = red[i & 1];
        if (lane < CL)
#pragma unroll
            for (int j = 0; j < WIDTH; j += 4) *reinterpret_cast<f32x4*>(&buf[wave][cl][j]) = f32x4{sum[j], sum[j + 1], sum[j + 2], sum[j + 3]};
        __syncthreads();
#pragma unroll
        for (int j = 0; j < WIDTH; j += 4) {
            f32x4 part[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) part[w] = *reinterpret_cast<const f32x4*>(&buf[w][cl][j]);
            part[0] = (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
            for (int n = 0; n < 4; ++n) sum[j + n] = part[0][n];
        }
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
            for (int j = 0; j < CV; ++j) y[(long long)c.step(p, i) * p.ys.t + j] = from_f32<T>(out[j]);
    }
    if (rg == 0 && on)
        for (long long t = c.len; t < p.T; ++t)
#pragma unroll
            for (int j = 0; j < CV; ++j) y[t * p.ys.t + j] = from_f32<T>(0.f);
    if (!p.last || !on) return;
#pragma unroll
    for (int n = 0; n < NR; ++n) {
        const int row = rg + n * RG;
        if (row < p.dk) store_f32<float, CV>(p.last + state + (long long)row * p.dv, s[n]);
    }
}

}  // namespace pdw
