// The logistic function and what is built from it, for the gated residual (row_norm.h) and the gated recurrence (scan.h).
#pragma once
#include "common.h"

namespace pdw {

enum : int { kActNone = 0, kActSigmoid = 1, kActSilu = 2 };

// exp(-v) for v >= 0.  v * log2(e) is rounded once, which alone would be v * 2^-24 of the result; the remainder of that product
// (from the fused multiply-add, and of log2(e) itself) goes back in by exp2(t + d) = exp2(t) (1 + d ln 2).
__device__ __forceinline__ float exp_neg(float v) {
    constexpr float kLog2e = 1.44269504f, kLog2eLow = 1.92596299e-8f, kLn2 = 0.693147181f;
    const float t = -v * kLog2e;
    const float d = __builtin_fmaf(-v, kLog2e, -t) - v * kLog2eLow;
    const float e = __builtin_amdgcn_exp2f(t);
    return v < 100.f ? __builtin_fmaf(e, d * kLn2, e) : 0.f;   // (past 100 nothing of it is left, and inf - inf would be NaN)
}

// a = sigmoid(g) and m = 1 - a = sigmoid(-g), both to full precision: with e = exp(-|g|) they are 1 / (1 + e) and e / (1 + e),
// whichever way round, so neither is a difference and nothing overflows (g = +-inf gives 1 and 0).
__device__ __forceinline__ void sigmoid_pair(float g, float& a, float& m) {
    const float e = exp_neg(fabsf(g));
    const float q = 1.f + e;
    float r = __builtin_amdgcn_rcpf(q);
    r = __builtin_fmaf(__builtin_fmaf(-q, r, 1.f), r, r);      // one Newton step: 1 ulp -> correctly rounded but for a few cases
    const float s = e * r;
    const bool pos = g >= 0.f;
    a = pos ? r : s, m = pos ? s : r;
    if (g != g) a = m = g;
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

}  // namespace pdw
