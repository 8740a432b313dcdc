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
// The kernels are bound by memory: they read each tensor once and write each once.  A row belongs to TPR neighbouring lanes (a
// power of two up to a wavefront, so that several short rows share one, or whole wavefronts), each holding NCH pieces of VEC
// channels (16 bytes) in registers from the load to the store, so the sums over a row are a few lane exchanges and the
// variance is taken from the centred values, in fp32.  Everything that is one value a channel (weights, scale, column sums) stays
// in the lane's registers while its workgroup walks over a segment of rows.
//
// The backward of a residual with its next norm behind 4096 channels (two pieces a lane in 16 bits, four in fp32) is the exception: its
// arrays take more than the 256 registers, and go through scratch memory.  Six tensors of 134 MB each: 4096 channels 147 us
// in bf16 and 142 in fp32 (5.5 and 5.7 TB/s), 8192 channels 211 and 302 (3.8 and 2.7).
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
    unsigned first;                                      // the launch's first workgroup (launch_parts)
    int act, kind, kind2;
    int gate_rows;                                       // 0: no gate; 1: a row an image; 2: a row a row
    float eps;
};

// A row segment: a workgroup has rows [r0, r1) of image `image`.
__device__ __forceinline__ void row_segment(const RowArgs& p, long long& r0, long long& r1, long long& image) {
    const unsigned block = p.first + blockIdx.x;
    image = block / (unsigned)p.S;
    const long long s = block - image * p.S, first = image * p.P;
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
        const int lanes = TPR > 64 ? (int)blockDim.x : TPR;
#pragma unroll
        for (int n = 0; n < NCH; ++n) {
            const int c = (n * lanes + lane) * VEC;
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

template <typename P, int N>
__device__ __forceinline__ void copy_row(P (&to)[N], const P (&from)[N]) {
#pragma unroll
    for (int n = 0; n < N; ++n) to[n] = from[n];
}

// Sum over lanes l, l ^ CTRL pattern within 16 lanes, in the VALU (data-parallel primitives).
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
    const int o = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true);
    return v + __builtin_bit_cast(float, o);
}

// Sum of lanes l and l ^ 16, and l ^ 32: the exchange of two rows of 16 lanes, and of the halves, leaves one side's values in one register
// and the other side's in the other.
__device__ __forceinline__ float swap_add16(float v) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const unsigned a = r[0], b = r[1];   // (a bit cast of an element would take the first one both times)
    return __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
}
__device__ __forceinline__ float swap_add32(float v) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const unsigned a = r[0], b = r[1];   // (a bit cast of an element would take the first one both times)
    return __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
}

// Sums of N values over the lanes of a row, in every one of them.  Rows of several wavefronts go through LDS, two buffers in turn
// (`flip`), so that one barrier a sum is enough; slots of wavefronts that there are not hold 0 (row_red_clear), so that all are read
// at once.
struct RowRed {
    float v[2][2][16];
};
template <int TPR>
__device__ __forceinline__ void row_red_clear(RowRed& red) {
    if constexpr (TPR > 64) {
        if (threadIdx.x < 64) red.v[threadIdx.x >> 5][threadIdx.x >> 4 & 1][threadIdx.x & 15] = 0.f;
        __syncthreads();
    }
}
template <int TPR, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], RowRed& red, int& flip) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = dpp_add<0xB1>(v[i]);    // quad permutation 1 0 3 2
        v[i] = dpp_add<0x4E>(v[i]);    // quad permutation 2 3 0 1
        v[i] = dpp_add<0x141>(v[i]);   // mirrored within 8
        if constexpr (TPR >= 16) v[i] = dpp_add<0x140>(v[i]);   // mirrored within 16
        if constexpr (TPR >= 32) v[i] = swap_add16(v[i]);
        if constexpr (TPR >= 64) v[i] = swap_add32(v[i]);
    }
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) red.v[flip][i][threadIdx.x >> 6] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float* r = red.v[flip][i];
            float s[TPR / 64];
#pragma unroll
            for (int w = 0; w < TPR / 64; ++w) s[w] = r[w];
#pragma unroll
            for (int h = TPR / 128; h > 0; h /= 2)
#pragma unroll
                for (int w = 0; w < h; ++w) s[w] += s[w + h];
            v[i] = s[0];
        }
        flip ^= 1;
    }
}

// Threads of a workgroup, at most: rows of up to a wavefront share one, longer ones have it to themselves and as many wavefronts as
// they need.
template <int TPR>
constexpr int row_threads(bool backward) {
    return TPR > 64 ? TPR : backward ? 512 : 256;
}

// 1 / sqrt(v).  The instruction takes subnormals for 0, whose result is infinity: with an eps of 0 rows below 1e-19 have such variances, which
// are taken 2^96 times as large.
__device__ __forceinline__ float reciprocal_root(float v) {
    const bool low = v < 0x1p-126f;
    return __builtin_amdgcn_rsqf(low ? v * 0x1p96f : v) * (low ? 0x1p48f : 1.f);
}

// Mean and reciprocal deviation of a row held in registers.
template <int VEC, int TPR, int NCH, typename COLS>
__device__ __forceinline__ float2 row_stats(const float (&v)[NCH][VEC], const COLS& cols, float inv_c, int kind, float eps,
                                            RowRed& red, int& flip) {
    float mean = 0.f;
    if (kind == kNormLayer) {
        float t[1] = {cols.sum([&](int n, int i) { return v[n][i]; })};
        row_sums<TPR, 1>(t, red, flip);
        mean = t[0] * inv_c;
    }
    float q[1] = {cols.sum([&](int n, int i) { return (v[n][i] - mean) * (v[n][i] - mean); })};
    row_sums<TPR, 1>(q, red, flip);
    return make_float2(mean, reciprocal_root(__builtin_fmaf(q[0], inv_c, eps)));
}

// x + f * norm(y), y's mean and reciprocal deviation in st.
__device__ __forceinline__ float residual_sum(float x, float f, float y, float2 st, float w, float b) {
    return __builtin_fmaf(f, __builtin_fmaf((y - st.x) * st.y, w, b), x);
}

// BRANCH: the residual (otherwise the norm by itself, of x); NEXT: the norm of the sum; FULL: a gate row for every row.
template <typename T, int VEC, int TPR, int NCH, bool RAG, bool BRANCH, bool NEXT, bool FULL>
__global__ __launch_bounds__(row_threads<TPR>(false)) void rows_fwd_k(RowArgs p) {
    constexpr int G = TPR > 64 ? 1 : row_threads<TPR>(false) / TPR;
    __shared__ RowRed red;
    int flip = 0;
    row_red_clear<TPR>(red);
    const int lane = TPR > 64 ? threadIdx.x : threadIdx.x % TPR, group = TPR > 64 ? 0 : threadIdx.x / TPR;
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
    Row xn, yn, gn;   // of the next row, on their way while this one is computed (behind the last one: the last again)
    auto load = [&](long long r) {
        if (BRANCH) cols.load((const T*)p.y + r * p.C, yn);
        if (FULL) cols.load((const T*)p.gate + r * p.ldg, gn);
        cols.load((const T*)p.x + r * p.C, xn);
    };
    if (r0 + group < r1) load(r0 + group);
    for (long long r = r0 + group; r < r1; r += G) {
        float v[NCH][VEC];
        Row xr, yr, gr;
        copy_row(xr, xn);
        if (BRANCH) copy_row(yr, yn);
        if (FULL) copy_row(gr, gn);
        load(r + G < r1 ? r + G : r);
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
    constexpr int THREADS = row_threads<TPR>(true), G = TPR > 64 ? 1 : THREADS / TPR;
    constexpr int SUMS = 2 * ((BRANCH ? 1 : 0) + (NEXT ? 1 : 0));
    __shared__ RowRed red;
    __shared__ float lds[TPR <= 64 ? THREADS / 64 * TPR * NCH * VEC : 1];
    int flip = 0;
    row_red_clear<TPR>(red);
    const int lane = TPR > 64 ? threadIdx.x : threadIdx.x % TPR, group = TPR > 64 ? 0 : threadIdx.x / TPR;
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
    Row gon, xn, gzn, yn, gn;   // of the next row, as in the forward
    float2 stn = make_float2(0.f, 1.f), st2n = stn;
    auto load = [&](long long r) {
        if (NEXT) st2n = reinterpret_cast<const float2*>(p.st2)[r];
        if (BRANCH && p.kind != kNormNone) stn = reinterpret_cast<const float2*>(p.st)[r];
        if (FULL) cols.load((const T*)p.gate + r * p.ldg, gn);
        if (BRANCH) cols.load((const T*)p.y + r * p.C, yn);
        if (NEXT) cols.load((const T*)p.x + r * p.C, xn), cols.load((const T*)p.gz + r * p.C, gzn);
        if (BRANCH) cols.load((const T*)p.go + r * p.C, gon);
    };
    if (r0 + group < r1) load(r0 + group);
    for (long long r = r0 + group; r < r1; r += G) {
        float go[NCH][VEC], nv[NCH][VEC], un[NCH][VEC];
        Row gor, xr, gzr, yr, gr;
        const float2 st = stn, st2 = st2n;
        if (FULL) copy_row(gr, gn);
        if (BRANCH) copy_row(yr, yn), copy_row(gor, gon);
        if (NEXT) copy_row(xr, xn), copy_row(gzr, gzn);
        load(r + G < r1 ? r + G : r);
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
            float t[2] = {cols.sum([&](int n, int i) { return un[n][i] * nv[n][i]; }), cols.sum([&](int n, int i) { return un[n][i]; })};
            row_sums<TPR, 2>(t, red, flip);
            const float a1 = t[0] * inv_c, a0 = p.kind2 == kNormLayer ? t[1] * inv_c : 0.f;
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
                float t[2] = {cols.sum([&](int n, int i) { return un[n][i] * nv[n][i]; }), cols.sum([&](int n, int i) { return un[n][i]; })};
                row_sums<TPR, 2>(t, red, flip);
                a1 = t[0] * inv_c, a0 = p.kind == kNormLayer ? t[1] * inv_c : 0.f;
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
    float* out = p.parts + (long long)(p.first + blockIdx.x) * SUMS * p.C;
    if (BRANCH) cols_out<VEC, TPR, NCH>(s1, cols, p.C, out, lds), cols_out<VEC, TPR, NCH>(s0, cols, p.C, out + p.C, lds);
    if (NEXT) {
        out += BRANCH ? 2 * p.C : 0;
        cols_out<VEC, TPR, NCH>(s1n, cols, p.C, out, lds), cols_out<VEC, TPR, NCH>(s0n, cols, p.C, out + p.C, lds);
    }
}

template <typename T, int VEC, int TPR, int NCH, bool RAG, bool BRANCH, bool NEXT, bool FULL>
void rows_pass(const RowArgs& p, unsigned grid, bool backward, hipStream_t s) {
    int threads = row_threads<TPR>(backward);
    if (TPR > 64) threads = ((p.C + VEC - 1) / VEC + 64 * NCH - 1) / (64 * NCH) * 64;
    RowArgs q = p;
    launch_parts(grid, threads, [&](long long first, unsigned n) {
        q.first = (unsigned)first;
        if (backward) rows_bwd_k<T, VEC, TPR, NCH, RAG, BRANCH, NEXT, FULL><<<n, threads, 0, s>>>(q);
        else rows_fwd_k<T, VEC, TPR, NCH, RAG, BRANCH, NEXT, FULL><<<n, threads, 0, s>>>(q);
    });
}

template <typename T, int VEC, int TPR, int NCH, bool RAG>
void rows_kind(const RowArgs& p, unsigned grid, bool backward, hipStream_t s) {
    const bool branch = p.y != nullptr, next = p.kind2 != kNormNone, full = p.gate_rows == 2;
    if (!branch) rows_pass<T, VEC, TPR, NCH, RAG, false, true, false>(p, grid, backward, s);
    else if (next && full) rows_pass<T, VEC, TPR, NCH, RAG, true, true, true>(p, grid, backward, s);
    else if (next) rows_pass<T, VEC, TPR, NCH, RAG, true, true, false>(p, grid, backward, s);
    else if (full) rows_pass<T, VEC, TPR, NCH, RAG, true, false, true>(p, grid, backward, s);
    else rows_pass<T, VEC, TPR, NCH, RAG, true, false, false>(p, grid, backward, s);
}

template <typename T, int VEC, int TPR, int NCH>
void rows_launch(const RowArgs& p, unsigned grid, bool backward, hipStream_t s) {
    if (VEC > 1 && p.C % VEC) rows_kind<T, VEC, TPR, NCH, (VEC > 1)>(p, grid, backward, s);
    else rows_kind<T, VEC, TPR, NCH, false>(p, grid, backward, s);
}

// Lanes of a row: one piece of 16 bytes each, in a part of a wavefront or in as many wavefronts as that takes, up to eight (0 here;
// behind 4096 channels, in fp32 2048, several pieces).  The backward of a gated residual with its next norm, [4,64,64,1152] fp16: 24
// channels a lane in one wavefront 227 us (430 registers), eight in three wavefronts 84, four in five 104 (the wavefronts wait for each
// other twice a row).
template <typename T>
int row_lanes(int C) {
    constexpr int V = 16 / sizeof(T);
    if (C < V) return 8;
    const int n = (C + V - 1) / V;
    return n <= 8 ? 8 : n <= 16 ? 16 : n <= 32 ? 32 : n <= 64 ? 64 : 0;
}

template <typename T>
void rows_dispatch(const RowArgs& p, unsigned grid, bool backward, hipStream_t s) {
    constexpr int V = 16 / sizeof(T);
    if (p.C < V) return rows_launch<T, 1, 8, 1>(p, grid, backward, s);
    switch (row_lanes<T>(p.C)) {
        case 8: return rows_launch<T, V, 8, 1>(p, grid, backward, s);
        case 16: return rows_launch<T, V, 16, 1>(p, grid, backward, s);
        case 32: return rows_launch<T, V, 32, 1>(p, grid, backward, s);
        case 64: return rows_launch<T, V, 64, 1>(p, grid, backward, s);
    }
    if (p.C <= 512 * V) rows_launch<T, V, 512, 1>(p, grid, backward, s);
    else if (p.C <= 1024 * V) rows_launch<T, V, 512, 2>(p, grid, backward, s);
    else if constexpr (sizeof(T) == 4) rows_launch<T, V, 512, 4>(p, grid, backward, s);
}

}  // namespace pdw
