// The logistic function and what is built from it, for the gated residual (row_norm.h) and the gated recurrence (scan.h).
#pragma once
#include "common.h"

namespace pdw {

enum : int { kActNone = 0, kActSigmoid = 1, kActSilu = 2 };

// a = sigmoid(g) and m = 1 - a = sigmoid(-g): with e = exp(-|g|) they are 1 / (1 + e) and e / (1 + e), whichever way round, so
// neither is a difference and nothing overflows (g = +-inf gives 1 and 0, NaN both NaN).  The larger is good to 2 u (u = 2^-24), the
// smaller to (|g| + 4) u of itself, which is less than u of the larger: |g| log2(e) is rounded, so e is off by |g| u, and what that
// moves a and m by is a m |g| u < u / 4.  (Taking the product's remainder along and a Newton step behind the reciprocal, both measured,
// changed no result's distance from the exact one and cost the recurrence a third of its instructions.)
__device__ __forceinline__ void sigmoid_pair(float g, float& a, float& m) {
    const float e = __builtin_amdgcn_exp2f(-fabsf(g) * 1.44269504f);
    const float r = __builtin_amdgcn_rcpf(1.f + e);
    const float s = e * r;
    const bool pos = g >= 0.f;
    a = pos ? r : s, m = pos ? s : r;
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
