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
// power of two up to a wavefront, so that several short rows share one, or whole wavefronts), each holding NCH pieces of VEC
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
    const void *go, *gz;                                 // gradients of out and next
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
    typedef Piece<T, VEC> Row[NCH];
    int at[NCH];   // first channel of a piece (0 where the row has none: the lane reads along and stores nothing)
    int own[NCH];  // channels of it before this one are another lane's too
    bool on[NCH];

    __device__ __forceinline__ RowCols(int lane, int C) {
#pragma unroll
        for (int n = 0; n < NCH; ++n) {
            const int c = (n * TPR + lane) * VEC;
            on[n] = c < C;
            at[n] = on[n] ? c : 0, own[n] = 0;
            if (RAG && on[n] && c + VEC > C) at[n] = C - VEC, own[n] = c - at[n];
        }
    }
    __device__ __forceinline__ bool mine(int n, int i) const { return on[n] && (!RAG || i >= own[n]); }

    // A sum over a lane's channels: f(n, i) of each that is its own.  (By pieces where a piece is whole: one selection for VEC values.)
    template <typename F>
    __device__ __forceinline__ float sum(F f) const {
        float s = 0.f;
#pragma unroll
        for (int n = 0; n < NCH; ++n) {
            float q = 0.f;
#pragma unroll
            for (int i = 0; i < VEC; ++i) q += !RAG || i >= own[n] ? f(n, i) : 0.f;
            s += on[n] ? q : 0.f;
        }
        return s;
    }
    // Every load is made, without a condition, so that all of a row's are on their way together.
    __device__ __forceinline__ void load(const T* row, Row& r) const {
#pragma unroll
        for (int n = 0; n < NCH; ++n) r[n] = load_any<T, VEC>(row + at[n]);
    }
    __device__ __forceinline__ void load_or(const T* row, float otherwise, Row& r) const {
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

// Sums of two values over the TPR lanes of a row, in every one of them.  Rows of several wavefronts go through LDS, two buffers in turn
// (`flip`), so that one barrier a sum is enough.
template <int TPR>
__device__ __forceinline__ void row_sum2(float& a, float& b, float2 (*red)[16], int& flip) {
    auto step = [&](auto f) { a = f(a), b = f(b); };
    step([](float v) { return dpp_add<0xB1>(v); });    // quad permutation 1 0 3 2
    step([](float v) { return dpp_add<0x4E>(v); });    // quad permutation 2 3 0 1
    step([](float v) { return dpp_add<0x141>(v); });   // mirrored within 8
    if constexpr (TPR >= 16) step([](float v) { return dpp_add<0x140>(v); });   // mirrored within 16
    if constexpr (TPR >= 32) step([](float v) { return v + __shfl_xor(v, 16); });
    if constexpr (TPR >= 64) step([](float v) { return v + __shfl_xor(v, 32); });
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63) == 0) red[flip][threadIdx.x >> 6] = make_float2(a, b);
        __syncthreads();
        a = b = 0.f;
#pragma unroll
        for (int w = 0; w < TPR / 64; ++w) a += red[flip][w].x, b += red[flip][w].y;
        flip ^= 1;
    }
}

// Threads of a workgroup: rows of up to a wavefront share one, longer ones have it to themselves.
template <int TPR>
constexpr int row_threads(bool backward) {
    return TPR > 64 ? TPR : backward ? 512 : 256;
}

// Mean and reciprocal deviation of a row held in registers.
template <int VEC, int TPR, int NCH, typename COLS>
__device__ __forceinline__ float2 row_stats(const float (&v)[NCH][VEC], const COLS& cols, float inv_c, int kind, float eps,
                                            float2 (*red)[16], int& flip) {
    float mean = 0.f, zero = 0.f;
    if (kind == kNormLayer) {
        mean = cols.sum([&](int n, int i) { return v[n][i]; });
        row_sum2<TPR>(mean, zero, red, flip);
        mean *= inv_c;
    }
    float q = cols.sum([&](int n, int i) { return (v[n][i] - mean) * (v[n][i] - mean); });
    row_sum2<TPR>(q, zero, red, flip);
    return make_float2(mean, __builtin_amdgcn_rsqf(__builtin_fmaf(q, inv_c, eps)));
}

// x + f * norm(y), y's mean and reciprocal deviation in st.
__device__ __forceinline__ float residual_sum(float x, float f, float y, float2 st, float w, float b) {
    return __builtin_fmaf(f, __builtin_fmaf((y - st.x) * st.y, w, b), x);
}

// BRANCH: the residual (otherwise the norm by itself, of x); NEXT: the norm of the sum; FULL: a gate row for every row.
template <typename T, int VEC, int TPR, int NCH, bool RAG, bool BRANCH, bool NEXT, bool FULL>
__global__ __launch_bounds__(row_threads<TPR>(false)) void rows_fwd_k(RowArgs p) {
    constexpr int G = row_threads<TPR>(false) / TPR;
    __shared__ float2 red[2][16];
    int flip = 0;
    const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
    const RowCols<T, VEC, TPR, NCH, RAG> cols(lane, p.C);
    typedef typename RowCols<T, VEC, TPR, NCH, RAG>::Row Row;
    long long r0, r1, image;
    row_segment(p, r0, r1, image);
    const float inv_c = 1.f / (float)p.C;
    Row w, b, w2, b2;
    float f[NCH][VEC];   // scale, and the gate's row where an image has one
    if (BRANCH) {
        Row sc, g;
        cols.load_or((const T*)p.w, 1.f, w), cols.load_or((const T*)p.b, 0.f, b), cols.load_or((const T*)p.scale, 1.f, sc);
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
        float v[NCH][VEC];
        Row xr, yr, gr;
        if (BRANCH) cols.load((const T*)p.y + r * p.C, yr);
        if (FULL) cols.load((const T*)p.gate + r * p.ldg, gr);
        cols.load((const T*)p.x + r * p.C, xr);
        if (BRANCH) {
#pragma unroll
            for (int n = 0; n < NCH; ++n)
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[n][i] = to_f32(yr[n].v[i]);
            float2 st = make_float2(0.f, 1.f);
            if (p.kind != kNormNone) st = row_stats<VEC, TPR, NCH>(v, cols, inv_c, p.kind, p.eps, red, flip);
            if (p.st && lane == 0) reinterpret_cast<float2*>(p.st)[r] = st;
            float a[NCH][VEC];
            if (FULL) gate_acts(gr, p.act, a);
#pragma unroll
            for (int n = 0; n < NCH; ++n) {
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    v[n][i] = residual_sum(to_f32(xr[n].v[i]), FULL ? f[n][i] * a[n][i] : f[n][i], v[n][i], st, to_f32(w[n].v[i]),
                                           to_f32(b[n].v[i]));
                cols.store((T*)p.out + r * p.C, n, v[n]);
            }
        } else {
#pragma unroll
            for (int n = 0; n < NCH; ++n)
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[n][i] = to_f32(xr[n].v[i]);
        }
        if (NEXT) {
            const float2 st = row_stats<VEC, TPR, NCH>(v, cols, inv_c, p.kind2, p.eps, red, flip);
            if (p.st2 && lane == 0) reinterpret_cast<float2*>(p.st2)[r] = st;
#pragma unroll
            for (int n = 0; n < NCH; ++n) {
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    v[n][i] = __builtin_fmaf((v[n][i] - st.x) * st.y, to_f32(w2[n].v[i]), to_f32(b2[n].v[i]));
                cols.store((T*)p.next + r * p.C, n, v[n]);
            }
        }
    }
}

// Column sums of a workgroup: over its row groups (lanes of a wavefront first, then the wavefronts through LDS), and out.
template <int VEC, int TPR, int NCH, typename COLS>
__device__ __forceinline__ void cols_out(float (&acc)[NCH][VEC], const COLS& cols, int C, float* __restrict__ out, float* lds) {
    constexpr int THREADS = row_threads<TPR>(true), WAVES = THREADS / 64;
    if constexpr (TPR < 64) {
#pragma unroll
        for (int n = 0; n < NCH; ++n)
#pragma unroll
            for (int i = 0; i < VEC; ++i)
#pragma unroll
                for (int d = TPR; d < 64; d *= 2) acc[n][i] += __shfl_xor(acc[n][i], d);
    }
    if constexpr (TPR > 64) {
#pragma unroll
        for (int n = 0; n < NCH; ++n)
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (cols.mine(n, i)) out[cols.at[n] + i] = acc[n][i];
    } else {
        constexpr int W = TPR * NCH * VEC;   // lds[WAVES][W]
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
        for (int c = threadIdx.x; c < C; c += THREADS) {
            float s = 0.f;
#pragma unroll
            for (int w = 0; w < WAVES; w += 2) s += lds[w * W + c] + lds[(w + 1) * W + c];
            out[c] = s;
        }
    }
}

template <typename T, int VEC, int TPR, int NCH, bool RAG, bool BRANCH, bool NEXT, bool FULL>
__global__ __launch_bounds__(row_threads<TPR>(true)) void rows_bwd_k(RowArgs p) {
    constexpr int THREADS = row_threads<TPR>(true), G = THREADS / TPR;
    constexpr int SUMS = 2 * ((BRANCH ? 1 : 0) + (NEXT ? 1 : 0));
    __shared__ float2 red[2][16];
    __shared__ float lds[TPR <= 64 ? THREADS / 64 * TPR * NCH * VEC : 1];
    int flip = 0;
    const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
    const RowCols<T, VEC, TPR, NCH, RAG> cols(lane, p.C);
    typedef typename RowCols<T, VEC, TPR, NCH, RAG>::Row Row;
    long long r0, r1, image;
    row_segment(p, r0, r1, image);
    const float inv_c = 1.f / (float)p.C;
    Row w, b, sc, w2;
    float f[NCH][VEC];   // scale, and the gate's row where an image has one
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
    for (long long r = r0 + group; r < r1; r += G) {
        float go[NCH][VEC], nv[NCH][VEC], un[NCH][VEC];
        Row gor, xr, gzr, yr, gr;
        float2 st = make_float2(0.f, 1.f), st2 = st;
        if (NEXT) st2 = reinterpret_cast<const float2*>(p.st2)[r];
        if (BRANCH && p.kind != kNormNone) st = reinterpret_cast<const float2*>(p.st)[r];
        if (FULL) cols.load((const T*)p.gate + r * p.ldg, gr);
        if (BRANCH) cols.load((const T*)p.y + r * p.C, yr);
        if (NEXT) cols.load((const T*)p.x + r * p.C, xr), cols.load((const T*)p.gz + r * p.C, gzr);
        if (BRANCH) cols.load((const T*)p.go + r * p.C, gor);
        float a[NCH][VEC], slope[NCH][VEC];
        if (FULL) gate_acts_slopes(gr, p.act, a, slope);
        if (NEXT) {
#pragma unroll
            for (int n = 0; n < NCH; ++n)
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float gz = to_f32(gzr[n].v[i]);
                    float v = to_f32(xr[n].v[i]);
                    if (BRANCH)   // the sum as the forward had it
                        v = residual_sum(v, FULL ? f[n][i] * a[n][i] : f[n][i], to_f32(yr[n].v[i]), st, to_f32(w[n].v[i]),
                                         to_f32(b[n].v[i]));
                    nv[n][i] = (v - st2.x) * st2.y;
                    un[n][i] = gz * to_f32(w2[n].v[i]);
                    s1n[n][i] = __builtin_fmaf(gz, nv[n][i], s1n[n][i]), s0n[n][i] += gz;
                }
            float a1 = cols.sum([&](int n, int i) { return un[n][i] * nv[n][i]; });
            float a0 = cols.sum([&](int n, int i) { return un[n][i]; });
            row_sum2<TPR>(a1, a0, red, flip);
            a1 *= inv_c, a0 = p.kind2 == kNormLayer ? a0 * inv_c : 0.f;
#pragma unroll
            for (int n = 0; n < NCH; ++n) {
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    go[n][i] = __builtin_fmaf(st2.y, un[n][i] - a0 - nv[n][i] * a1, BRANCH ? to_f32(gor[n].v[i]) : 0.f);
                if (p.gx) cols.store((T*)p.gx + r * p.C, n, go[n]);
            }
        } else {
#pragma unroll
            for (int n = 0; n < NCH; ++n)
#pragma unroll
                for (int i = 0; i < VEC; ++i) go[n][i] = to_f32(gor[n].v[i]);
        }
        if (BRANCH) {
#pragma unroll
            for (int n = 0; n < NCH; ++n) {
                float gg[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    nv[n][i] = (to_f32(yr[n].v[i]) - st.x) * st.y;
                    float fi = f[n][i], u = go[n][i];
                    if (FULL) {
                        gg[i] = u * fi * slope[n][i] * __builtin_fmaf(nv[n][i], to_f32(w[n].v[i]), to_f32(b[n].v[i]));
                        fi *= a[n][i], u *= a[n][i];
                    }
                    un[n][i] = go[n][i] * fi * to_f32(w[n].v[i]);
                    s1[n][i] = __builtin_fmaf(u, nv[n][i], s1[n][i]), s0[n][i] += u;
                }
                if (FULL && p.ggate) cols.store((T*)p.ggate + r * p.C, n, gg);
            }
            float a1 = 0.f, a0 = 0.f;
            if (p.kind != kNormNone) {
                a1 = cols.sum([&](int n, int i) { return un[n][i] * nv[n][i]; });
                a0 = cols.sum([&](int n, int i) { return un[n][i]; });
                row_sum2<TPR>(a1, a0, red, flip);
                a1 *= inv_c, a0 = p.kind == kNormLayer ? a0 * inv_c : 0.f;
            }
            if (p.gy) {
#pragma unroll
                for (int n = 0; n < NCH; ++n) {
                    float o[VEC];
#pragma unroll
                    for (int i = 0; i < VEC; ++i) o[i] = st.y * (un[n][i] - a0 - nv[n][i] * a1);
                    cols.store((T*)p.gy + r * p.C, n, o);
                }
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

template <typename T, int VEC, int TPR, int NCH, bool RAG, bool BRANCH, bool NEXT, bool FULL>
void rows_pass(const RowArgs& p, unsigned grid, bool backward, hipStream_t s) {
    if (backward) rows_bwd_k<T, VEC, TPR, NCH, RAG, BRANCH, NEXT, FULL><<<grid, row_threads<TPR>(true), 0, s>>>(p);
    else rows_fwd_k<T, VEC, TPR, NCH, RAG, BRANCH, NEXT, FULL><<<grid, row_threads<TPR>(false), 0, s>>>(p);
}

template <typename T, int VEC, int TPR, int NCH, bool RAG>
void rows_launch(const RowArgs& p, unsigned grid, bool backward, hipStream_t s) {
    const bool branch = p.y != nullptr, next = p.kind2 != kNormNone, full = p.gate_rows == 2;
    if (!branch) rows_pass<T, VEC, TPR, NCH, RAG, false, true, false>(p, grid, backward, s);
    else if (next && full) rows_pass<T, VEC, TPR, NCH, RAG, true, true, true>(p, grid, backward, s);
    else if (next) rows_pass<T, VEC, TPR, NCH, RAG, true, true, false>(p, grid, backward, s);
    else if (full) rows_pass<T, VEC, TPR, NCH, RAG, true, false, true>(p, grid, backward, s);
    else rows_pass<T, VEC, TPR, NCH, RAG, true, false, false>(p, grid, backward, s);
}

// Lanes of a row: as few as hold it in one piece each, so that a wavefront's loads cover whole rows and a lane's column sums stay
// few (with three pieces a lane the backward of a gated residual had 430 registers, one wavefront on a SIMD and 227 us at
// [4,64,64,1152] fp16).
template <typename T>
int row_lanes(int C) {
    constexpr int V = 16 / sizeof(T);
    if (C < V) return 8;
    const int n = (C + V - 1) / V;
    return n <= 8 ? 8 : n <= 16 ? 16 : n <= 32 ? 32 : n <= 64 ? 64 : n <= 128 ? 128 : n <= 192 ? 192 : n <= 256 ? 256 : n <= 512 ? 512 : 1024;
}

template <typename T>
void rows_dispatch(const RowArgs& p, unsigned grid, bool backward, hipStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const int n = (p.C + V - 1) / V;
#define PDW_ROWS(tpr, nch)                                                                       \
    (p.C % V ? rows_launch<T, V, tpr, nch, true>(p, grid, backward, s) : rows_launch<T, V, tpr, nch, false>(p, grid, backward, s))
    if (p.C < V) return rows_launch<T, 1, 8, 1, false>(p, grid, backward, s);
    switch (row_lanes<T>(p.C)) {
        case 8: return PDW_ROWS(8, 1);
        case 16: return PDW_ROWS(16, 1);
        case 32: return PDW_ROWS(32, 1);
        case 64: return PDW_ROWS(64, 1);
        case 128: return PDW_ROWS(128, 1);
        case 192: return PDW_ROWS(192, 1);
        case 256: return PDW_ROWS(256, 1);
        case 512: return PDW_ROWS(512, 1);
    }
    if (n <= 1024) PDW_ROWS(1024, 1);
    else if constexpr (sizeof(T) == 4) PDW_ROWS(1024, 2);
#undef PDW_ROWS
}

}  // namespace pdw
