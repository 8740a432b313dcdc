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

// The same for a gate: silu(v) = v a and its slope a (1 + v m) would be made large again far below zero by a of 2^-126 (-4 at the lowest
// bfloat16, a mask's usual value).  So v is limited instead, to where e is infinite, a 0 and all results 0, at v = -inf too; the product for m
// is clamped to [0, 1], which takes infinity times 0 to 0 and is part of the multiplication.  (NaN passes: through v and a.)  Between -87.3 and the
// limit a may be flushed: silu and its slope are under 88 e^-87 < 2^-118 there.  As many instructions as sigmoid_pair.  The residual of
// [4,64,64,1152] fp16 with a silu gate a value, forward and backward: 126.2 us; with comparisons and selections of 0 behind
// sigmoid_pair 128.6, with a minimum for m 127.7, with a branch for each activation in the forward 127.8.
__device__ __forceinline__ void gate_parts(float v, float& limited, float& a, float& m) {
    limited = __builtin_elementwise_maximum(v, -126.f);
    const float e = __builtin_amdgcn_exp2f(limited * -1.44269504f);
    a = __builtin_amdgcn_rcpf(1.f + e);
    m = __builtin_amdgcn_fmed3f(e * a, 0.f, 1.f);
}

// act(v), and act'(v)
__device__ __forceinline__ float gate_act(float v, int act) {
    if (act == kActNone) return v;
    float s, q, m;
    gate_parts(v, s, q, m);
    return act == kActSigmoid ? q : s * q;
}

__device__ __forceinline__ void gate_act_slope(float v, int act, float& f, float& slope) {
    f = v, slope = 1.f;
    if (act == kActNone) return;
    float s, q, m;
    gate_parts(v, s, q, m);
    if (act == kActSigmoid) f = q, slope = q * m;
    else f = s * q, slope = q * __builtin_fmaf(s, m, 1.f);
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
            float s, q, m;
            gate_parts(a[n][i], s, q, m);
            a[n][i] = act == kActSilu ? s * q : q;
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
                float s, m;
                gate_parts(a[n][i], s, a[n][i], m);
                slope[n][i] = a[n][i] * m;
            }
        return;
    }
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            float s, q, m;
            gate_parts(a[n][i], s, q, m);
            slope[n][i] = q * __builtin_fmaf(s, m, 1.f);
            a[n][i] = s * q;
        }
}

}  // namespace pdw
