// Norms over the channels of rows, and the gated residual that closes a block, forward and backward.
//
//   norm      n = (v - mean) * rstd, rstd = 1 / sqrt(mean (v - mean)^2 + eps)  (rms: mean = 0);  norm(v) = n w + b
//   residual  out = x + scale * act(gate) * norm(y),  and the next block's norm of out where it is wanted
//   backward  of a norm, with t its output's gradient and u = t w:  rstd (u - mean(u) - n mean(u n))  (rms: without mean(u));
//             of its weight and bias the sums over rows of t n and t.  Of the residual, with g = out's gradient:
//             S1 = sum g act n and S0 = sum g act give scale's gradient w S1 + b S0, w's scale S1 and b's scale S0, so two column
//             sums serve all three; with a gate row for each image the sums are kept by image and give the gate's gradient too.
//             The backward makes out again from x and y (y it reads anyway): read back as it was stored, its rounding would be in
//             every gradient (0.0027 off the exact ones in bf16, 0.0017 this way; one rounding of a result is 0.0017).
//
// Every kernel is bound by memory: it reads each tensor once and writes each once.  A row belongs to TPR neighbouring lanes (a
// power of two up to a wavefront, so that several short rows share one, or a workgroup of 256), each holding NCH pieces of VEC
// channels (16 bytes) in registers from the load to the store, so the sums over a row are a few lane exchanges and the
// variance is taken from the centred values, in fp32.  Everything that is one value a channel (weights, scale, column sums) stays
// in the lane's registers while its workgroup walks over a segment of rows.
//
// Channel counts that are no multiple of VEC (RAG): the row's last piece begins VEC before its end and overlaps the one before
// it; the overlapped values are left out of every sum and are stored twice with the same bits.  Rows that do not start on 16 bytes
// are loaded and stored as they lie (global memory takes any alignment here).
#pragma once
#include "common.h"
#include "gate_math.h"

namespace pdw {

enum : int { kNormNone = 0, kNormRms = 1, kNormLayer = 2 };

struct RowArgs {
    const void *x, *y, *gate, *scale, *w, *b, *w2, *b2;  // forward inputs
    void *out, *next;
    float *st, *st2;                                     // (mean, rstd) of each row: of y, and of the next norm's input
    const void *go, *gz;                                 // gradients of out and next (either may be null)
    void *gx, *gy, *ggate;
    float* parts;                                        // column sums of a segment: [segment][sums][C]
    long long N, P, L;                                   // rows; rows of an image; rows of a segment
    long long ldg;                                       // elements between gate rows
    int C, S;                                            // channels; segments of an image
    int act, kind, kind2;
    int gate_rows;                                       // 0: no gate; 1: a row an image; 2: a row a row
    float eps;
};

// A row segment: workgroup blockIdx.x has rows [r0, r1) of image `image`.
__device__ __forceinline__ void row_segment(const RowArgs& p, long long& r0, long long& r1, long long& image) {
    image = blockIdx.x / (unsigned)p.S;
    const long long s = blockIdx.x - image * p.S, first = image * p.P;
    r0 = first + s * p.L;
    r1 = r0 + p.L < first + p.P ? r0 + p.L : first + p.P;
}

template <typename T, int VEC>
struct Piece {
    T v[VEC];
};

// A piece moves as one access of its size, wherever it lies (as an array of 16-bit values a store of it comes out in halves).
template <int BYTES>
struct AccessOf;
template <>
struct AccessOf<2> {
    typedef unsigned short type;
};
template <>
struct AccessOf<4> {
    typedef unsigned type;
};
template <>
struct AccessOf<8> {
    typedef unsigned type __attribute__((ext_vector_type(2)));
};
template <>
struct AccessOf<16> {
    typedef unsigned type __attribute__((ext_vector_type(4)));
};
template <typename T, int VEC>
struct Access {
    typedef typename AccessOf<sizeof(T) * VEC>::type word;
    typedef word type __attribute__((aligned(sizeof(T)), may_alias));
};

template <typename T, int VEC>
__device__ __forceinline__ Piece<T, VEC> load_any(const T* p) {
    typename Access<T, VEC>::word w = *reinterpret_cast<const typename Access<T, VEC>::type*>(p);
    return __builtin_bit_cast(Piece<T, VEC>, w);
}

template <typename T, int VEC>
__device__ __forceinline__ Piece<T, VEC> round_piece(const float (&v)[VEC]) {
    Piece<T, VEC> r;
#pragma unroll
    for (int i = 0; i < VEC; ++i) r.v[i] = from_f32<T>(v[i]);
    return r;
}

template <typename T, int VEC>
__device__ __forceinline__ void store_piece(T* p, const Piece<T, VEC>& r) {
    *reinterpret_cast<typename Access<T, VEC>::type*>(p) = __builtin_bit_cast(typename Access<T, VEC>::word, r);
}

template <typename T, int VEC>
__device__ __forceinline__ void store_any(T* p, const float (&v)[VEC]) {
    store_piece<T, VEC>(p, round_piece<T, VEC>(v));
}

// A lane's pieces of a row.
template <typename T, int VEC, int TPR, int NCH, bool RAG>
struct RowCols {
    int at[NCH];   // first channel of a piece
    int own[NCH];  // channels of it before this one are another lane's too
    bool on[NCH];

    __device__ __forceinline__ RowCols(int lane, int C) {
#pragma unroll
        for (int n = 0; n < NCH; ++n) {
            const int c = (n * TPR + lane) * VEC;
            on[n] = c < C;
            at[n] = c, own[n] = 0;
            if (RAG && on[n] && c + VEC > C) at[n] = C - VEC, own[n] = c - at[n];
        }
    }
    __device__ __forceinline__ bool mine(int n, int i) const { return on[n] && (!RAG || i >= own[n]); }

    // Pieces of a row; zeros where the row has none (their values are stored nowhere, and every sum leaves them out).
    __device__ __forceinline__ void load(const T* row, Piece<T, VEC> (&r)[NCH]) const {
#pragma unroll
        for (int n = 0; n < NCH; ++n) {
            if (on[n]) r[n] = load_any<T, VEC>(row + at[n]);
            else
#pragma unroll
                for (int i = 0; i < VEC; ++i) r[n].v[i] = from_f32<T>(0.f);
        }
    }
    __device__ __forceinline__ void load_or(const T* row, float otherwise, Piece<T, VEC> (&r)[NCH]) const {
        if (row) return load(row, r);
#pragma unroll
        for (int n = 0; n < NCH; ++n)
#pragma unroll
            for (int i = 0; i < VEC; ++i) r[n].v[i] = from_f32<T>(otherwise);
    }
    __device__ __forceinline__ void store(T* row, int n, const float (&v)[VEC]) const {
        if (on[n]) store_any<T, VEC>(row + at[n], v);
    }
};

// Sum over lanes l, l ^ CTRL pattern within 16 lanes, in the VALU (data-parallel primitives).
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
    const int o = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true);
    return v + __builtin_bit_cast(float, o);
}

// Sums of two values over the TPR lanes of a row, in every one of them.  `red`: LDS of a row as wide as the workgroup, used
// in turn (`flip`) so that one barrier a sum is enough.
template <int TPR>
__device__ __forceinline__ void row_sum2(float& a, float& b, float2 (*red)[4], int& flip) {
    auto step = [&](auto f) { a = f(a), b = f(b); };
    step([](float v) { return dpp_add<0xB1>(v); });    // quad permutation 1 0 3 2
    step([](float v) { return dpp_add<0x4E>(v); });    // quad permutation 2 3 0 1
    step([](float v) { return dpp_add<0x141>(v); });   // mirrored within 8
    if constexpr (TPR >= 16) step([](float v) { return dpp_add<0x140>(v); });   // mirrored within 16
    if constexpr (TPR >= 32) step([](float v) { return v + __shfl_xor(v, 16); });
    if constexpr (TPR >= 64) step([](float v) { return v + __shfl_xor(v, 32); });
    if constexpr (TPR == 256) {
        if ((threadIdx.x & 63) == 0) red[flip][threadIdx.x >> 6] = make_float2(a, b);
        __syncthreads();
        const float2 *r = red[flip];
        a = (r[0].x + r[1].x) + (r[2].x + r[3].x), b = (r[0].y + r[1].y) + (r[2].y + r[3].y);
        flip ^= 1;
    }
}

// Mean and reciprocal deviation of a row held in registers.
template <int VEC, int TPR, int NCH, typename COLS>
__device__ __forceinline__ void row_stats(const float (&v)[NCH][VEC], const COLS& cols, int C, int kind, float eps, float& mean,
                                          float& rstd, float2 (*red)[4], int& flip) {
    mean = 0.f;
    float s = 0.f, zero = 0.f;
    if (kind == kNormLayer) {
#pragma unroll
        for (int n = 0; n < NCH; ++n)
#pragma unroll
            for (int i = 0; i < VEC; ++i) s += cols.mine(n, i) ? v[n][i] : 0.f;
        row_sum2<TPR>(s, zero, red, flip);
        mean = s / (float)C;
    }
    float q = 0.f;
#pragma unroll
    for (int n = 0; n < NCH; ++n)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float d = v[n][i] - mean;
            q += cols.mine(n, i) ? d * d : 0.f;
        }
    row_sum2<TPR>(q, zero, red, flip);
    rstd = 1.f / sqrtf(q / (float)C + eps);
}

// x + f * norm(y), y's mean and reciprocal deviation in st.
__device__ __forceinline__ float residual_sum(float x, float f, float y, float2 st, float w, float b) {
    return __builtin_fmaf(f, __builtin_fmaf((y - st.x) * st.y, w, b), x);
}

// BRANCH: the residual (otherwise the norm by itself, of x); NEXT: the norm of the sum.
template <typename T, int VEC, int TPR, int NCH, bool RAG, bool BRANCH, bool NEXT>
__global__ __launch_bounds__(256) void rows_fwd_k(RowArgs p) {
    constexpr int G = 256 / TPR;
    __shared__ float2 red[2][4];
    int flip = 0;
    const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
    const RowCols<T, VEC, TPR, NCH, RAG> cols(lane, p.C);
    long long r0, r1, image;
    row_segment(p, r0, r1, image);
    typedef Piece<T, VEC> Row[NCH];
    Row w, b, sc, w2, b2;
    float f[NCH][VEC];   // scale, and the gate's row where an image has one
    if (BRANCH) {
        cols.load_or((const T*)p.w, 1.f, w), cols.load_or((const T*)p.b, 0.f, b), cols.load_or((const T*)p.scale, 1.f, sc);
        Row g;
        if (p.gate_rows == 1) cols.load((const T*)p.gate + image * p.ldg, g);
#pragma unroll
        for (int n = 0; n < NCH; ++n)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                f[n][i] = to_f32(sc[n].v[i]);
                if (p.gate_rows == 1) f[n][i] *= gate_act(to_f32(g[n].v[i]), p.act);
            }
    }
    if (NEXT) cols.load_or((const T*)p.w2, 1.f, w2), cols.load_or((const T*)p.b2, 0.f, b2);
    for (long long r = r0 + group; r < r1; r += G) {
        float v[NCH][VEC], mean, rstd;
        Row xr, yr, gr;
        cols.load((const T*)p.x + r * p.C, xr);
        if (BRANCH) {
            cols.load((const T*)p.y + r * p.C, yr);
            if (p.gate_rows == 2) cols.load((const T*)p.gate + r * p.ldg, gr);
#pragma unroll
            for (int n = 0; n < NCH; ++n)
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[n][i] = to_f32(yr[n].v[i]);
            mean = 0.f, rstd = 1.f;
            if (p.kind != kNormNone) row_stats<VEC, TPR, NCH>(v, cols, p.C, p.kind, p.eps, mean, rstd, red, flip);
            if (p.st && lane == 0) reinterpret_cast<float2*>(p.st)[r] = make_float2(mean, rstd);
#pragma unroll
            for (int n = 0; n < NCH; ++n) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    float fi = f[n][i];
                    if (p.gate_rows == 2) fi *= gate_act(to_f32(gr[n].v[i]), p.act);
                    v[n][i] = residual_sum(to_f32(xr[n].v[i]), fi, v[n][i], make_float2(mean, rstd), to_f32(w[n].v[i]), to_f32(b[n].v[i]));
                }
                cols.store((T*)p.out + r * p.C, n, v[n]);
            }
        } else {
#pragma unroll
            for (int n = 0; n < NCH; ++n)
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[n][i] = to_f32(xr[n].v[i]);
        }
        if (NEXT) {
            row_stats<VEC, TPR, NCH>(v, cols, p.C, p.kind2, p.eps, mean, rstd, red, flip);
            if (p.st2 && lane == 0) reinterpret_cast<float2*>(p.st2)[r] = make_float2(mean, rstd);
#pragma unroll
            for (int n = 0; n < NCH; ++n) {
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    v[n][i] = __builtin_fmaf((v[n][i] - mean) * rstd, to_f32(w2[n].v[i]), to_f32(b2[n].v[i]));
                cols.store((T*)p.next + r * p.C, n, v[n]);
            }
        }
    }
}

// Column sums of a workgroup: over its row groups (lanes of a wavefront first, then the four wavefronts through LDS), and out.
template <int VEC, int TPR, int NCH, typename COLS>
__device__ __forceinline__ void cols_out(float (&acc)[NCH][VEC], const COLS& cols, int C, float* __restrict__ out, float* lds) {
    if constexpr (TPR < 64) {
#pragma unroll
        for (int n = 0; n < NCH; ++n)
#pragma unroll
            for (int i = 0; i < VEC; ++i)
#pragma unroll
                for (int d = TPR; d < 64; d *= 2) acc[n][i] += __shfl_xor(acc[n][i], d);
    }
    if constexpr (TPR == 256) {
#pragma unroll
        for (int n = 0; n < NCH; ++n)
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (cols.mine(n, i)) out[cols.at[n] + i] = acc[n][i];
    } else {
        constexpr int W = TPR * NCH * VEC;   // lds[4][W]
        const int wave = threadIdx.x >> 6;
        __syncthreads();
        if ((threadIdx.x & 63) < TPR) {
#pragma unroll
            for (int n = 0; n < NCH; ++n)
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    if (cols.mine(n, i)) lds[wave * W + cols.at[n] + i] = acc[n][i];
        }
        __syncthreads();
        for (int c = threadIdx.x; c < C; c += 256)
            out[c] = (lds[c] + lds[W + c]) + (lds[2 * W + c] + lds[3 * W + c]);
    }
}

template <typename T, int VEC, int TPR, int NCH, bool RAG, bool BRANCH, bool NEXT>
__global__ __launch_bounds__(256) void rows_bwd_k(RowArgs p) {
    constexpr int G = 256 / TPR;
    constexpr int SUMS = 2 * ((BRANCH ? 1 : 0) + (NEXT ? 1 : 0));
    __shared__ float2 red[2][4];
    __shared__ float lds[TPR < 256 ? 4 * TPR * NCH * VEC : 1];
    int flip = 0;
    const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
    const RowCols<T, VEC, TPR, NCH, RAG> cols(lane, p.C);
    long long r0, r1, image;
    row_segment(p, r0, r1, image);
    typedef Piece<T, VEC> Row[NCH];
    Row w, b, sc, w2;
    float f[NCH][VEC];
    float s1[NCH][VEC], s0[NCH][VEC], s1n[NCH][VEC], s0n[NCH][VEC];
#pragma unroll
    for (int n = 0; n < NCH; ++n)
#pragma unroll
        for (int i = 0; i < VEC; ++i) s1[n][i] = s0[n][i] = s1n[n][i] = s0n[n][i] = 0.f;
    if (BRANCH) {
        cols.load_or((const T*)p.w, 1.f, w), cols.load_or((const T*)p.b, 0.f, b), cols.load_or((const T*)p.scale, 1.f, sc);
        Row g;
        if (p.gate_rows == 1) cols.load((const T*)p.gate + image * p.ldg, g);
#pragma unroll
        for (int n = 0; n < NCH; ++n)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                f[n][i] = to_f32(sc[n].v[i]);
                if (p.gate_rows == 1) f[n][i] *= gate_act(to_f32(g[n].v[i]), p.act);
            }
    }
    if (NEXT) cols.load_or((const T*)p.w2, 1.f, w2);
    const float inv_c = 1.f / (float)p.C;
    for (long long r = r0 + group; r < r1; r += G) {
        float go[NCH][VEC], nv[NCH][VEC], un[NCH][VEC];
        Row gor, xr, gzr, yr, gr;
        cols.load_or(p.go ? (const T*)p.go + r * p.C : nullptr, 0.f, gor);
        if (NEXT) cols.load((const T*)p.x + r * p.C, xr), cols.load_or(p.gz ? (const T*)p.gz + r * p.C : nullptr, 0.f, gzr);
        if (BRANCH) {
            cols.load((const T*)p.y + r * p.C, yr);
            if (p.gate_rows == 2) cols.load((const T*)p.gate + r * p.ldg, gr);
        }
        float2 sty = make_float2(0.f, 1.f);
        if (BRANCH && p.kind != kNormNone) sty = reinterpret_cast<const float2*>(p.st)[r];
#pragma unroll
        for (int n = 0; n < NCH; ++n)
#pragma unroll
            for (int i = 0; i < VEC; ++i) go[n][i] = to_f32(gor[n].v[i]);
        if (NEXT) {
            const float2 st = reinterpret_cast<const float2*>(p.st2)[r];
            float a1 = 0.f, a0 = 0.f;
#pragma unroll
            for (int n = 0; n < NCH; ++n)
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float gz = to_f32(gzr[n].v[i]);
                    float v = to_f32(xr[n].v[i]);
                    if (BRANCH) {   // the sum as the forward had it
                        float fi = f[n][i];
                        if (p.gate_rows == 2) fi *= gate_act(to_f32(gr[n].v[i]), p.act);
                        v = residual_sum(v, fi, to_f32(yr[n].v[i]), sty, to_f32(w[n].v[i]), to_f32(b[n].v[i]));
                    }
                    nv[n][i] = (v - st.x) * st.y;
                    un[n][i] = gz * to_f32(w2[n].v[i]);
                    const bool mine = cols.mine(n, i);
                    a1 += mine ? un[n][i] * nv[n][i] : 0.f, a0 += mine ? un[n][i] : 0.f;
                    s1n[n][i] = __builtin_fmaf(gz, nv[n][i], s1n[n][i]), s0n[n][i] += gz;
                }
            row_sum2<TPR>(a1, a0, red, flip);
            a1 *= inv_c, a0 = p.kind2 == kNormLayer ? a0 * inv_c : 0.f;
#pragma unroll
            for (int n = 0; n < NCH; ++n) {
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    go[n][i] = __builtin_fmaf(st.y, un[n][i] - a0 - nv[n][i] * a1, go[n][i]);
                if (p.gx) cols.store((T*)p.gx + r * p.C, n, go[n]);
            }
        }
        if (BRANCH) {
            const float2 st = sty;
            float a1 = 0.f, a0 = 0.f;
#pragma unroll
            for (int n = 0; n < NCH; ++n) {
                float gg[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    nv[n][i] = (to_f32(yr[n].v[i]) - st.x) * st.y;
                    float fi = f[n][i], u = go[n][i];
                    if (p.gate_rows == 2) {
                        float act, slope;
                        gate_act_slope(to_f32(gr[n].v[i]), p.act, act, slope);
                        gg[i] = u * fi * slope * __builtin_fmaf(nv[n][i], to_f32(w[n].v[i]), to_f32(b[n].v[i]));
                        fi *= act, u *= act;
                    }
                    un[n][i] = go[n][i] * fi * to_f32(w[n].v[i]);
                    const bool mine = cols.mine(n, i);
                    a1 += mine ? un[n][i] * nv[n][i] : 0.f, a0 += mine ? un[n][i] : 0.f;
                    s1[n][i] = __builtin_fmaf(u, nv[n][i], s1[n][i]), s0[n][i] += u;
                }
                if (p.gate_rows == 2 && p.ggate) cols.store((T*)p.ggate + r * p.C, n, gg);
            }
            if (p.kind != kNormNone) row_sum2<TPR>(a1, a0, red, flip);
            a1 *= inv_c, a0 = p.kind == kNormLayer ? a0 * inv_c : 0.f;
            if (p.kind == kNormNone) a1 = 0.f;
#pragma unroll
            for (int n = 0; n < NCH; ++n) {
                float o[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) o[i] = st.y * (un[n][i] - a0 - nv[n][i] * a1);
                if (p.gy) cols.store((T*)p.gy + r * p.C, n, o);
            }
        }
    }
    if (!p.parts) return;
    float* out = p.parts + (long long)blockIdx.x * SUMS * p.C;
    if (BRANCH) cols_out<VEC, TPR, NCH>(s1, cols, p.C, out, lds), cols_out<VEC, TPR, NCH>(s0, cols, p.C, out + p.C, lds);
    if (NEXT) {
        out += BRANCH ? 2 * p.C : 0;
        cols_out<VEC, TPR, NCH>(s1n, cols, p.C, out, lds), cols_out<VEC, TPR, NCH>(s0n, cols, p.C, out + p.C, lds);
    }
}

template <typename T, int VEC, int TPR, int NCH, bool RAG>
void rows_launch(const RowArgs& p, unsigned grid, bool backward, hipStream_t s) {
    const bool branch = p.y != nullptr, next = p.kind2 != kNormNone;
#define PDW_ROWS(k) k<<<grid, 256, 0, s>>>(p)
    if (!backward) {
        if (branch && next) PDW_ROWS((rows_fwd_k<T, VEC, TPR, NCH, RAG, true, true>));
        else if (branch) PDW_ROWS((rows_fwd_k<T, VEC, TPR, NCH, RAG, true, false>));
        else PDW_ROWS((rows_fwd_k<T, VEC, TPR, NCH, RAG, false, true>));
    } else {
        if (branch && next) PDW_ROWS((rows_bwd_k<T, VEC, TPR, NCH, RAG, true, true>));
        else if (branch) PDW_ROWS((rows_bwd_k<T, VEC, TPR, NCH, RAG, true, false>));
        else PDW_ROWS((rows_bwd_k<T, VEC, TPR, NCH, RAG, false, true>));
    }
#undef PDW_ROWS
}

// Lanes of a row: as few as hold it in one piece each, so that a wavefront's loads cover whole rows; past a wavefront up to
// four pieces, then a workgroup.
template <typename T>
int row_lanes(int C) {
    constexpr int V = 16 / sizeof(T);
    if (C < V) return 8;
    const int n = (C + V - 1) / V;
    return n <= 8 ? 8 : n <= 16 ? 16 : n <= 32 ? 32 : n <= 256 ? 64 : 256;
}

template <typename T>
void rows_dispatch(const RowArgs& p, unsigned grid, bool backward, hipStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const int n = (p.C + V - 1) / V;
#define PDW_ROWS(tpr, nch)                                                                       \
    (p.C % V ? rows_launch<T, V, tpr, nch, true>(p, grid, backward, s) : rows_launch<T, V, tpr, nch, false>(p, grid, backward, s))
    if (p.C < V) rows_launch<T, 1, 8, 1, false>(p, grid, backward, s);
    else if (n <= 8) PDW_ROWS(8, 1);
    else if (n <= 16) PDW_ROWS(16, 1);
    else if (n <= 32) PDW_ROWS(32, 1);
    else if (n <= 64) PDW_ROWS(64, 1);
    else if (n <= 128) PDW_ROWS(64, 2);
    else if (n <= 192) PDW_ROWS(64, 3);
    else if (n <= 256) PDW_ROWS(64, 4);
    else if (n <= 512) PDW_ROWS(256, 2);
    else if (n <= 1024) PDW_ROWS(256, 4);
    else if constexpr (sizeof(T) == 4) PDW_ROWS(256, 8);
#undef PDW_ROWS
}

}  // namespace pdw
