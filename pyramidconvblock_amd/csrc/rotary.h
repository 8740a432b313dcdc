// Norms of the rows of heads (queries, keys) with the rotation by positions in the same pass, forward and backward.
//
//   n = x  (none),   x r w,  r = 1 / sqrt(mean x^2 + eps) (rms) or 1 / sqrt(sum x^2 + eps) (l2);    of n's d channels the first 2 P are P pairs
//   (a, b): halves (i, P + i) or neighbours (2 i, 2 i + 1), and pair i becomes (a cos t - b sin t, b cos t + a sin t), t = position frequency_i,
//   the position along the axis that the pair belongs to.  Backward: the gradient is turned back, then u = g w and
//   gx = r (u - x r mean(u x r)) (l2: the sum instead of the mean), gw = sum over rows of g x r.  The backward makes r again from x.
//
// Bound by memory: a row's channels stay in registers between one load and one store.  A unit is 2 VEC channels, VEC whole pairs (or channels
// behind the pairs); a row has up to LPR lanes with a unit each, so its sum is a few exchanges in the vector unit.  A workgroup has TT tokens:
// it makes their cosines and sines once, into LDS, for all heads of q and k.  An angle counts in turns and in 64 bits up to the nearest
// quarter: what is left is below 1/8 of a turn and off by some 2^-53 of the angle itself (2^-24 of a turn at position 2^31, nothing that counts at 2^20);
// cosine and sine of that are their series.
//
// Measured: 50176 tokens of 8 and 4 heads of 64 in bf16 (rms, three axes) 37 us forward, 154 MB moved, 4.1 TB/s, vector instructions issued in 73 % of the time;
// backward 68 + 7 us, 232 MB, 3.4 TB/s, 60 %.  16384 tokens of 9 and 9 heads of 128 in fp16, 32 pairs turned, no norm: 37 us forward, 42 backward, 151 MB
// each.  3136 tokens of 4 and 4 heads of 32: 7 us, angles and latencies.
#pragma once
#include "common.h"
#include "row_norm.h"

namespace pdw {

constexpr int kRotaryMaxDim = 256;
enum : int { kRotaryNone = 0, kRotaryRms = 1, kRotaryL2 = 2 };
enum : int { kPositionGrid = 0, kPositionI32 = 1, kPositionI64 = 2, kPositionF32 = 3 };

struct RotaryArgs {
    const void* x[2];             // q and k; element (token, head, i) at token * xt + head * xh + i
    long long xt[2], xh[2];
    void* y[2];                   // dense; backward: gx (or null)
    const void* gy[2];            // dense
    const void* w[2];             // [d], or null
    float* parts;                 // [workgroup][2][d]: sums for the weights' gradients, or null
    const void* positions;        // [rows][axes]
    const float* frequencies;     // [P] in radians, or null: `turns`
    long long N, np;              // tokens; rows of positions
    int grid[3], ends[3];         // extents of the last axes; pairs before the end of each axis' section
    int heads[2], d, P, axes, kind, neighbours, pkind, TT;
    float eps;
    double turns[kRotaryMaxDim / 2];   // frequencies in turns
};

// cos and sin of a number of turns
__device__ __forceinline__ float2 cos_sin_turns(double t) {
    t -= rint(t);
    t *= 4.0;
    const double n = rint(t);
    const float x = (float)((t - n) * 1.5707963267948966);   // up to pi / 4
    const float z = x * x;
    const float s = x * (1.f + z * (-1.f / 6 + z * (1.f / 120 + z * (-1.f / 5040 + z * (1.f / 362880)))));
    const float c = 1.f + z * (-0.5f + z * (1.f / 24 + z * (-1.f / 720 + z * (1.f / 40320 + z * (-1.f / 3628800)))));
    const int q = (int)n & 3;
    const float a = q & 1 ? s : c, b = q & 1 ? c : s;
    return make_float2(q == 1 || q == 2 ? -a : a, q & 2 ? -b : b);
}

template <int LPR>
__device__ __forceinline__ float lanes_sum(float v) {
    if constexpr (LPR >= 2) v = dpp_add<0xB1>(v);
    if constexpr (LPR >= 4) v = dpp_add<0x4E>(v);
    if constexpr (LPR >= 8) v = dpp_add<0x141>(v);
    if constexpr (LPR >= 16) v = dpp_add<0x140>(v);
    if constexpr (LPR >= 32) v = swap_add16(v);
    if constexpr (LPR >= 64) v = swap_add32(v);
    return v;
}

// UPL units a lane (more than one only where VEC = 1 and a row has more than 64 pairs).
template <typename T, int VEC, int LPR, int UPL, bool BWD>
__global__ __launch_bounds__(256) void rotary_k(RotaryArgs p) {
    constexpr int GROUPS = 256 / LPR;
    extern __shared__ __align__(16) float2 cs[];   // [TT][P]
    const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
    const int rot = p.P / VEC, units = rot + (p.d - 2 * p.P) / (2 * VEC) + (VEC == 1 && (p.d & 1));
    // where a lane's two pieces lie; `odd`: the last channel of an odd d has no partner
    int at[UPL], to[UPL], pair[UPL];
    bool on[UPL], turn[UPL], odd[UPL];
#pragma unroll
    for (int n = 0; n < UPL; ++n) {
        const int u = lane + n * LPR;
        on[n] = u < units, turn[n] = u < rot;
        const int v = on[n] ? u : 0;
        pair[n] = turn[n] ? v * VEC : 0;
        if (turn[n] && !p.neighbours) at[n] = v * VEC, to[n] = p.P + v * VEC;
        else at[n] = 2 * VEC * v, to[n] = at[n] + VEC;   // (2 P = 2 VEC rot channels lie before the first unit that is not turned)
        if (!on[n]) at[n] = 0, to[n] = VEC == 1 && p.d == 1 ? 0 : VEC;
        odd[n] = on[n] && to[n] >= p.d;
        if (odd[n]) to[n] = at[n];
    }
    float acc[2][UPL][2 * VEC];
    if constexpr (BWD) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int n = 0; n < UPL; ++n)
#pragma unroll
                for (int i = 0; i < 2 * VEC; ++i) acc[s][n][i] = 0.f;
    }
    const long long blocks = (p.N + p.TT - 1) / p.TT;
    for (long long b = blockIdx.x; b < blocks; b += gridDim.x) {
        const long long t0 = b * p.TT;
        const int nt = (int)(p.N - t0 < p.TT ? p.N - t0 : p.TT);
        if (b != blockIdx.x) __syncthreads();
        for (int e = threadIdx.x; e < nt * p.P; e += 256) {
            const int tok = e / p.P, i = e - tok * p.P;
            const int axis = i >= p.ends[0] ? i >= p.ends[1] ? 2 : 1 : 0;
            const double f = p.frequencies ? (double)p.frequencies[i] * 0.15915494309189535 : p.turns[i];
            const long long t = t0 + tok;
            double pos;
            if (p.pkind == kPositionGrid) {
                const long long row = t / p.grid[2], plane = row / p.grid[1];
                const int last = (int)(t - row * p.grid[2]), mid = (int)(row - plane * p.grid[1]), first = (int)(plane % p.grid[0]);
                const int which = axis + 3 - p.axes;
                pos = which == 2 ? last : which == 1 ? mid : first;
            } else {
                const long long j = t % p.np * p.axes + axis;
                pos = p.pkind == kPositionI32   ? (double)((const int*)p.positions)[j]
                      : p.pkind == kPositionI64 ? (double)((const long long*)p.positions)[j]
                                                : (double)((const float*)p.positions)[j];
            }
            cs[e] = cos_sin_turns(pos * f);
        }
        __syncthreads();
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int H = p.heads[s];
            if (!H || (BWD && !p.y[s] && !p.parts)) continue;
            float w[UPL][2 * VEC];
#pragma unroll
            for (int n = 0; n < UPL; ++n)
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    w[n][i] = p.w[s] ? to_f32(((const T*)p.w[s])[at[n] + i]) : 1.f;
                    w[n][VEC + i] = p.w[s] ? to_f32(((const T*)p.w[s])[to[n] + i]) : 1.f;
                }
            const int rows = nt * H;
            for (int r0 = 0; r0 < rows; r0 += GROUPS) {
                const bool live = r0 + group < rows;
                const int r = live ? r0 + group : rows - 1;
                const int tok = r / H, h = r - tok * H;
                const long long dense = ((t0 + tok) * H + h) * p.d;
                const T* x = (const T*)p.x[s] + (t0 + tok) * p.xt[s] + h * p.xh[s];
                // (all as they come: what is taken apart ahead of the next load is waited for there)
                typedef typename Access<T, VEC>::word word;
                typedef typename Access<T, VEC>::type any;
                word rx[UPL][2], rg[UPL][2];
                const bool normed = !BWD || p.kind != kRotaryNone;
#pragma unroll
                for (int n = 0; n < UPL; ++n)
                    if (normed) rx[n][0] = *reinterpret_cast<const any*>(x + at[n]), rx[n][1] = *reinterpret_cast<const any*>(x + to[n]);
                if constexpr (BWD) {
                    const T* gy = (const T*)p.gy[s] + dense;
#pragma unroll
                    for (int n = 0; n < UPL; ++n) rg[n][0] = *reinterpret_cast<const any*>(gy + at[n]), rg[n][1] = *reinterpret_cast<const any*>(gy + to[n]);
                }
                float v[UPL][2 * VEC], q[UPL][2 * VEC];   // x (then its norm); backward: the gradient
                float sum = 0.f;
                auto floats = [&](const word(&from)[2], int n, float(&o)[2 * VEC]) {
                    const Piece<T, VEC> a = __builtin_bit_cast(Piece<T, VEC>, from[0]), c = __builtin_bit_cast(Piece<T, VEC>, from[1]);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) o[i] = on[n] ? to_f32(a.v[i]) : 0.f, o[VEC + i] = on[n] && !odd[n] ? to_f32(c.v[i]) : 0.f;
                };
#pragma unroll
                for (int n = 0; n < UPL; ++n) {
                    if (normed) floats(rx[n], n, v[n]);
                    if constexpr (BWD) floats(rg[n], n, q[n]);
                }
                float rs = 1.f;
                const float part = p.kind == kRotaryRms ? 1.f / p.d : 1.f;
                if (p.kind != kRotaryNone) {
#pragma unroll
                    for (int n = 0; n < UPL; ++n)
#pragma unroll
                        for (int i = 0; i < 2 * VEC; ++i) sum = __builtin_fmaf(v[n][i], v[n][i], sum);
                    rs = reciprocal_root(lanes_sum<LPR>(sum) * part + p.eps);
                }
                float(&z)[UPL][2 * VEC] = BWD ? q : v;
                if constexpr (!BWD) {
#pragma unroll
                    for (int n = 0; n < UPL; ++n)
#pragma unroll
                        for (int i = 0; i < 2 * VEC; ++i) v[n][i] = v[n][i] * rs * w[n][i];
                }
#pragma unroll
                for (int n = 0; n < UPL; ++n) {
                    if (!turn[n]) continue;
                    const float2* c = cs + tok * p.P + pair[n];
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        const float2 t = c[i];
                        const float sn = BWD ? -t.y : t.y;
                        if (p.neighbours) {
                            const float a = z[n][2 * i], d = z[n][2 * i + 1];
                            z[n][2 * i] = a * t.x - d * sn, z[n][2 * i + 1] = d * t.x + a * sn;
                        } else {
                            const float a = z[n][i], d = z[n][VEC + i];
                            z[n][i] = a * t.x - d * sn, z[n][VEC + i] = d * t.x + a * sn;
                        }
                    }
                }
                if constexpr (BWD) {
                    if (p.kind != kRotaryNone) {
                        float dot = 0.f;
#pragma unroll
                        for (int n = 0; n < UPL; ++n)
#pragma unroll
                            for (int i = 0; i < 2 * VEC; ++i) {
                                v[n][i] *= rs;
                                if (live) acc[s][n][i] = __builtin_fmaf(q[n][i], v[n][i], acc[s][n][i]);
                                q[n][i] *= w[n][i];
                                dot = __builtin_fmaf(q[n][i], v[n][i], dot);
                            }
                        dot = lanes_sum<LPR>(dot) * part;
#pragma unroll
                        for (int n = 0; n < UPL; ++n)
#pragma unroll
                            for (int i = 0; i < 2 * VEC; ++i) q[n][i] = rs * __builtin_fmaf(-v[n][i], dot, q[n][i]);
                    }
                }
                if (live && p.y[s]) {
                    T* y = (T*)p.y[s] + dense;
#pragma unroll
                    for (int n = 0; n < UPL; ++n) {
                        if (!on[n]) continue;
                        float a[VEC], c[VEC];
#pragma unroll
                        for (int i = 0; i < VEC; ++i) a[i] = z[n][i], c[i] = z[n][VEC + i];
                        store_any<T, VEC>(y + at[n], a);
                        if (!odd[n]) store_any<T, VEC>(y + to[n], c);
                    }
                }
            }
        }
    }
    if constexpr (BWD) {
        if (!p.parts) return;
        // the groups' sums in a fixed order, through LDS
        float* red = (float*)cs;   // [GROUPS][d]
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            __syncthreads();
#pragma unroll
            for (int n = 0; n < UPL; ++n) {
                if (!on[n]) continue;
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    red[group * p.d + at[n] + i] = acc[s][n][i];
                    if (!odd[n]) red[group * p.d + to[n] + i] = acc[s][n][VEC + i];
                }
            }
            __syncthreads();
            for (int c = threadIdx.x; c < p.d; c += 256) {
                float sum = 0.f;
                for (int g = 0; g < GROUPS; ++g) sum += red[g * p.d + c];
                p.parts[((long long)blockIdx.x * 2 + s) * p.d + c] = sum;
            }
        }
    }
}

template <typename T, int VEC, int LPR, int UPL>
inline void rotary_shape_launch(const RotaryArgs& p, unsigned grid, bool backward, hipStream_t s) {
    size_t lds = (size_t)p.TT * p.P * sizeof(float2);
    const size_t red = (size_t)(256 / LPR) * p.d * sizeof(float);
    if (backward && p.parts && lds < red) lds = red;
    if (backward) rotary_k<T, VEC, LPR, UPL, true><<<grid, 256, lds, s>>>(p);
    else rotary_k<T, VEC, LPR, UPL, false><<<grid, 256, lds, s>>>(p);
}

// Channels of a piece: as many as 16 bytes hold, fewer where pairs or channels behind them do not come out in whole units.
template <typename T>
inline int rotary_vec(int d, int P) {
    for (int vec = 16 / (int)sizeof(T); vec >= 4; vec /= 2)
        if (P % vec == 0 && (d - 2 * P) % (2 * vec) == 0) return vec;
    return 1;
}
template <typename T>
inline int rotary_lanes(int d, int P) {
    const int vec = rotary_vec<T>(d, P), units = (d + 2 * vec - 1) / (2 * vec);
    int lanes = vec == 1 ? 64 : vec == 4 ? 2 : 1;
    while (lanes < units && lanes < 64) lanes *= 2;
    return lanes;
}

template <typename T>
inline void rotary_dispatch(const RotaryArgs& p, unsigned grid, bool backward, hipStream_t s) {
    const int vec = rotary_vec<T>(p.d, p.P), lanes = rotary_lanes<T>(p.d, p.P);
    if (vec == 1) return rotary_shape_launch<T, 1, 64, 2>(p, grid, backward, s);
    if (vec == 4) {
        if (lanes == 2) return rotary_shape_launch<T, 4, 2, 1>(p, grid, backward, s);
        if (lanes == 4) return rotary_shape_launch<T, 4, 4, 1>(p, grid, backward, s);
        if (lanes == 8) return rotary_shape_launch<T, 4, 8, 1>(p, grid, backward, s);
        if (lanes == 16) return rotary_shape_launch<T, 4, 16, 1>(p, grid, backward, s);
        return rotary_shape_launch<T, 4, 32, 1>(p, grid, backward, s);
    }
    if constexpr (sizeof(T) == 2) {
        if (lanes == 1) return rotary_shape_launch<T, 8, 1, 1>(p, grid, backward, s);
        if (lanes == 2) return rotary_shape_launch<T, 8, 2, 1>(p, grid, backward, s);
        if (lanes == 4) return rotary_shape_launch<T, 8, 4, 1>(p, grid, backward, s);
        if (lanes == 8) return rotary_shape_launch<T, 8, 8, 1>(p, grid, backward, s);
        return rotary_shape_launch<T, 8, 16, 1>(p, grid, backward, s);
    }
}

}  // namespace pdw
