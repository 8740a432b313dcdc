// The logistic function and what is built from it, for the gated residual (row_norm.h) and the gated recurrence (scan.h).
#pragma once
#include "common.h"

namespace pdw {

enum : int { kActNone = 0, kActSigmoid = 1, kActSilu = 2 };

// a = sigmoid(g) = 1 / (1 + e) and m = 1 - a = sigmoid(-g) = e / (1 + e) with e = exp(-g), so m is no difference.  e is limited to 2^126,
// from where a is 2^-126 instead of less (g = -inf: m = 1; g = inf: a = 1 and m = 0; NaN passes).  g log2(e) is rounded, so e is off
// by |g| u (u = 2^-24): that moves the smaller of a and m by that much of itself, and the larger by a m |g| u < u / 4.  (Taking the product's
// remainder along and a Newton step behind the reciprocal, both measured, changed no result's distance from the exact one and cost the
// recurrence a third of its instructions.)
__device__ __forceinline__ void sigmoid_pair(float g, float& a, float& m) {
    const float e = __builtin_amdgcn_exp2f(__builtin_elementwise_minimum(g * -1.44269504f, 126.f));
    a = __builtin_amdgcn_rcpf(1.f + e);
    m = e * a;
}

// act(v), and act'(v)
__device__ __forceinline__ float gate_act(float v, int act) {
    if (act == kActNone) return v;
    float q, m;
    sigmoid_pair(v, q, m);
    return act == kActSigmoid ? q : v * q;
}

__device__ __forceinline__ void gate_act_slope(float v, int act, float& f, float& slope) {
    f = v, slope = 1.f;
    if (act == kActNone) return;
    float q, m;
    sigmoid_pair(v, q, m);
    if (act == kActSigmoid) f = q, slope = q * m;
    else f = v * q, slope = q * __builtin_fmaf(v, m, 1.f);
}

// The same for a lane's pieces of a row (one branch for all of them).
template <typename P, int N, int VEC>
__device__ __forceinline__ void gate_acts(const P (&g)[N], int act, float (&a)[N][VEC]) {
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < VEC; ++i) a[n][i] = to_f32(g[n].v[i]);
    if (act == kActNone) return;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            float q, m;
            sigmoid_pair(a[n][i], q, m);
            a[n][i] = act == kActSilu ? a[n][i] * q : q;
        }
}

template <typename P, int N, int VEC>
__device__ __forceinline__ void gate_acts_slopes(const P (&g)[N], int act, float (&a)[N][VEC], float (&slope)[N][VEC]) {
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < VEC; ++i) a[n][i] = to_f32(g[n].v[i]), slope[n][i] = 1.f;
    if (act == kActNone) return;
    if (act == kActSigmoid) {
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                float m;
                sigmoid_pair(a[n][i], a[n][i], m);
                slope[n][i] = a[n][i] * m;
            }
        return;
    }
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            float q, m;
            sigmoid_pair(a[n][i], q, m);
            slope[n][i] = q * __builtin_fmaf(a[n][i], m, 1.f);
            a[n][i] *= q;
        }
}

}  // namespace pdw
