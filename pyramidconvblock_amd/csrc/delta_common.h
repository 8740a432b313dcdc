// The gated delta rule: what its kernels share.  (The mathematics: delta_fwd.h and delta_bwd.h.)
//
// Products run on the bf16 matrix cores whatever the tensors' type: a value is a sum of bf16 planes (the value rounded, what that left
// rounded, and so on), and a product of two such sums leaves out the products of planes that are below the result's precision.  What comes from
// the tensors takes as many planes as hold it exactly (1 for bf16, 2 for fp16, 3 for fp32); what was computed in fp32 (the chunk's triangular system,
// its solutions, states) takes 3 planes, 24 bits, where states come of it, which are results in 32 bits, and 2 planes, 2^-17 of a value, where
// it ends in results of 16 bits, and in the gradients of fp32 gates beside 16-bit tensors: those gradients hold some 17 bits of what they are sums of (off by 3e-6 to 8e-6 of
// their norm), more than the 8 or 11 that came in with dY, and a third plane would cost a launch that waits for LDS its second workgroup a compute unit.  Sums are the matrix
// cores' fp32.  So results are off by their own rounding and by little else (bf16, 32 x 3136 steps: 0.35 % are not the nearest value, and off by up to 1.11 half
// steps), where single bf16 operands had put 2^-9 of every intermediate into them; and fp32 takes 6 products of 16 cycles where the fp32 matrix
// instruction takes eight of 32.
//
// Fragments of the 16x16x32 instruction: lane l has row (column) l % 16 and 8 values along the inner axis.  A result has column l % 16 and
// rows 4 (l / 16) + r, so results turn into operands of a next product whose inner axis is their rows without an exchange of lanes: an inner
// axis of 32 is two tiles of 16 rows, value j of lane group g stands for row 16 (j / 4) + 4 g + j % 4 ("tile order"), and the other operand is
// read in that order too.
#pragma once
#include "common.h"
#include "row_norm.h"

namespace pdw {

constexpr int kDeltaChunk = 64;   // steps of a chunk
constexpr int kDeltaPad = 8;      // values behind an LDS row: rows of 16 values in a row stay on different banks

// Element (o, t, w, head, i) of a tensor is base[o * o + t * t + w * w + head * h + i].
struct DeltaStrides {
    long long o, t, w, h;
};

struct DeltaArgs {
    const void *q, *k, *v, *g, *b, *gy;
    DeltaStrides qs, ks, vs, gs, bs;
    DeltaStrides ys;                       // of y and gy
    void *y, *gq, *gk, *gv, *gg, *gb;      // gradients dense: [O][T][W][heads][..]
    DeltaStrides gqs, gvs, ggs;            // gqs of gq and gk, ggs of gg and gb
    const float *h0, *glast;               // [chain][dk][dv], or null (0)
    float *last, *gh0;                     // [chain][dk][dv], or null
    const int* lengths;                    // [O], or null (T)
    // between the kernels, by chain and chunk
    bf16_t *s0, *u, *ds1, *blocks;
    float *w, *ub, *du, *c0;
    struct DeltaGates* gates;
    bf16_t* maps;                          // by chain and segment: the map's matrix, and what it adds
    float* shifts;
    int T, NC, seg;                        // steps; chunks of a chain, of a segment
    int segments;
    int O, W, Hk, Hv, dk, dv, dvp;         // dvp: dv up to whole 32s
    int chains;                            // O * W * Hv, one state each
    long long first;                       // the launch's first workgroup (launch_parts)
    int reverse, logits, gates_f32;
    int vec;                               // bits: q, k, v, gy, y, gq and gk, gv lie in aligned rows of whole pieces of 8
    float scale;
};

enum : int { kVecQ = 1, kVecK = 2, kVecV = 4, kVecGy = 8, kVecY = 16, kVecGqk = 32, kVecGv = 64 };

// Planes of what states are made of: they are results in 32 bits.
constexpr int kChainPlanes = 3;

template <typename T>
struct DeltaPlanes;
template <>
struct DeltaPlanes<bf16_t> {
    static constexpr int kRaw = 1, kMade = 2;
};
template <>
struct DeltaPlanes<f16_t> {
    static constexpr int kRaw = 2, kMade = 2;
};
template <>
struct DeltaPlanes<float> {
    static constexpr int kRaw = 3, kMade = 3;
};

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <int NP>
struct Frag {   // inner axis of 32
    bf16x8 p[NP];
};
template <int NP>
struct Half {   // inner axis of 16: value j of lane group g is 4 g + j
    bf16x4 p[NP];
};

// c + a b: the products of planes i and j with i + j below N, by default the larger number of planes, the small ones first.  (N = 3 for products of
// tensors that states come of: of fp16's two planes each the last product is 2^-18.)
template <int N_ = 0, int NA, int NB>
__device__ __forceinline__ f32x4 mma(const Frag<NA>& a, const Frag<NB>& b, f32x4 c) {
    constexpr int N = N_ ? N_ : NA > NB ? NA : NB;
#pragma unroll
    for (int s = N - 1; s >= 0; --s)
#pragma unroll
        for (int i = 0; i <= s; ++i)
            if (i < NA && s - i < NB) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[i], b.p[s - i], c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ f32x4 mma16(bf16x4 a, bf16x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a), __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
}
template <int NA, int NB>
__device__ __forceinline__ f32x4 mma(const Half<NA>& a, const Half<NB>& b, f32x4 c) {
    constexpr int N = NA > NB ? NA : NB;
#pragma unroll
    for (int s = N - 1; s >= 0; --s)
#pragma unroll
        for (int i = 0; i <= s; ++i)
            if (i < NA && s - i < NB) c = mma16(a.p[i], b.p[s - i], c);
    return c;
}

// The same for several first operands, their products in turn: one waits for the last only when all have had theirs.
template <int R, int NA, int NB>
__device__ __forceinline__ void mma_rows(const Frag<NA> (&a)[R], const Frag<NB>& b, f32x4 (&c)[R]) {
    constexpr int N = NA > NB ? NA : NB;
#pragma unroll
    for (int s = N - 1; s >= 0; --s)
#pragma unroll
        for (int i = 0; i <= s; ++i)
            if (i < NA && s - i < NB) {
#pragma unroll
                for (int r = 0; r < R; ++r) c[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[r].p[i], b.p[s - i], c[r], 0, 0, 0);
            }
}
// The first planes.
template <int NP, int N>
__device__ __forceinline__ Frag<NP> planes(const Frag<N>& f) {
    Frag<NP> r;
#pragma unroll
    for (int p = 0; p < NP; ++p) r.p[p] = f.p[p];
    return r;
}

template <int NP>
__device__ __forceinline__ Half<NP> split(f32x4 v) {
    Half<NP> h;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
#pragma unroll
        for (int i = 0; i < 4; ++i) h.p[p][i] = (__bf16)v[i];
        if (p + 1 < NP) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] -= (float)h.p[p][i];
        }
    }
    return h;
}
// of a b, unrounded
template <int NP>
__device__ __forceinline__ Half<NP> split_product(f32x4 a, f32x4 b) {
    Half<NP> h;
    const f32x4 v = a * b;
    f32x4 rest;
#pragma unroll
    for (int i = 0; i < 4; ++i) h.p[0][i] = (__bf16)v[i], rest[i] = __builtin_fmaf(a[i], b[i], -(float)h.p[0][i]);
    const Half<NP - 1> more = split<NP - 1>(rest);
#pragma unroll
    for (int p = 1; p < NP; ++p) h.p[p] = more.p[p - 1];
    return h;
}
template <int NP>
__device__ __forceinline__ Frag<NP> join(const Half<NP>& a, const Half<NP>& b) {
    Frag<NP> f;
#pragma unroll
    for (int p = 0; p < NP; ++p) f.p[p] = __builtin_shufflevector(a.p[p], b.p[p], 0, 1, 2, 3, 4, 5, 6, 7);
    return f;
}
template <int NP>
__device__ __forceinline__ f32x4 sum_of(const Half<NP>& h) {
    f32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = (float)h.p[NP - 1][i];
#pragma unroll
        for (int p = NP - 2; p >= 0; --p) v[i] += (float)h.p[p][i];
    }
    return v;
}

// A uniform address and a lane's own bytes behind it: one addition less a load than with 64-bit lane addresses.
template <typename V>
__device__ __forceinline__ V load_at(const void* base, unsigned bytes) {
    return *reinterpret_cast<const V*>((const char*)base + bytes);
}
template <typename V>
__device__ __forceinline__ void store_at(void* base, unsigned bytes, V v) {
    *reinterpret_cast<V*>((char*)base + bytes) = v;
}

// The planes of 8 values of a tensor.
template <typename T, int NP>
__device__ __forceinline__ Frag<NP> planes_of(const T (&v)[8]) {
    Frag<NP> f;
    if constexpr (sizeof(T) == 2 && NP == 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f.p[0][i] = v[i];
    } else {
        float r[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = to_f32(v[i]);
#pragma unroll
        for (int p = 0; p < NP; ++p) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                f.p[p][i] = (__bf16)r[i];
                r[i] -= (float)f.p[p][i];
            }
        }
    }
    return f;
}

// The operand that turns a tile round: 1 where lane and value meet.  (Products by 1 and sums with 0: exact.)
__device__ __forceinline__ bf16x4 unit_half(int lane) {
    bf16x4 u;
#pragma unroll
    for (int j = 0; j < 4; ++j) u[j] = (__bf16)(4 * (lane >> 4) + j == (lane & 15) ? 1.f : 0.f);
    return u;
}
// A tile's plane, lane = column and values = rows, with lane = row and values = columns.
__device__ __forceinline__ bf16x4 turned(bf16x4 t, bf16x4 unit) {
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    const f32x4 r = mma16(t, unit, zero);
    bf16x4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = (__bf16)r[j];
    return o;
}

// A tile as it was made (lane = column, values = rows; 8 bytes a lane and plane, planes `plane` values apart) from LDS, with lane = row, values = columns:
// lane l of each 16 hands in column 4 g + l / 4, rows 4 (l % 4) .., and gets row l % 16, columns 4 g ...  (WIDTH: values between lanes' pieces.)
template <int NP, int WIDTH = 4>
__device__ __forceinline__ Half<NP> read_turned(const bf16_t* base, int plane, int lane) {
    typedef __attribute__((address_space(3))) s16x4 lds_t;
    const int i = lane & 15, from = (i & 3) * 16 + 4 * (lane >> 4) + (i >> 2);
    Half<NP> f;
#pragma unroll
    for (int p = 0; p < NP; ++p)
        f.p[p] = __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t*)(__attribute__((address_space(3))) void*)(base + p * plane + from * WIDTH)));
    return f;
}

// LDS rows of R values of planes: value i of row r of plane p at [p][r][i].
template <int NP, int ROWS, int R>
struct Rows {
    static constexpr int kStride = R + kDeltaPad, kPlane = ROWS * kStride, kValues = NP * kPlane;
    // 8 consecutive values of a lane's row: the inner axis in its own order (32 n + 8 g ..)
    static __device__ __forceinline__ Frag<NP> natural(const bf16_t* base, int row, int at, int lane) {
        Frag<NP> f;
#pragma unroll
        for (int p = 0; p < NP; ++p)
            f.p[p] = *reinterpret_cast<const bf16x8*>(base + p * kPlane + (row + (lane & 15)) * kStride + at + 8 * (lane >> 4));
        return f;
    }
    // in tile order
    static __device__ __forceinline__ Half<NP> half(const bf16_t* base, int row, int at, int lane) {
        Half<NP> f;
#pragma unroll
        for (int p = 0; p < NP; ++p)
            f.p[p] = *reinterpret_cast<const bf16x4*>(base + p * kPlane + (row + (lane & 15)) * kStride + at + 4 * (lane >> 4));
        return f;
    }
    static __device__ __forceinline__ Frag<NP> tiles(const bf16_t* base, int row, int at, int lane) {
        return join(half(base, row, at, lane), half(base, row, at + 16, lane));
    }
    // a tile (lane = column, values = rows) to its rows, turned
    static __device__ __forceinline__ void put_turned(bf16_t* base, int row, int at, const Half<NP>& h, bf16x4 unit, int lane) {
#pragma unroll
        for (int p = 0; p < NP; ++p)
            *reinterpret_cast<bf16x4*>(base + p * kPlane + (row + (lane & 15)) * kStride + at + 4 * (lane >> 4)) = turned(h.p[p], unit);
    }
    // lane = column `at` + l % 16, values = rows row + 4 g ..: every group of 16 lanes reads four rows of 16 values, transposed on the way
    static __device__ __forceinline__ Half<NP> down(const bf16_t* base, int row, int at, int lane) {
        typedef __attribute__((address_space(3))) s16x4 lds_t;
        Half<NP> f;
        const int i = lane & 15;
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            const bf16_t* q = base + p * kPlane + (row + 4 * (lane >> 4) + (i >> 2)) * kStride + at + 4 * (i & 3);
            f.p[p] = __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t*)(__attribute__((address_space(3))) void*)q));
        }
        return f;
    }
};

// Where a chain stands in its tensors.
struct DeltaChain {
    int o, w, hv, hk;
    int len;   // valid steps
    __device__ __forceinline__ DeltaChain(const DeltaArgs& p, int chain) {
        hv = chain % p.Hv;
        const int ow = chain / p.Hv;
        w = ow % p.W, o = ow / p.W;
        hk = hv / (p.Hv / p.Hk);
        len = p.T;
        if (p.lengths) {
            const int n = p.lengths[o];
            len = n < 0 ? 0 : n < len ? n : len;
        }
    }
    // The step at place i of the chain: from the end of what is valid with `reverse`, and places behind it for themselves.
    __device__ __forceinline__ int step(const DeltaArgs& p, int i) const { return p.reverse && i < len ? len - 1 - i : i; }
    __device__ __forceinline__ long long at(const DeltaStrides& s, int head) const { return o * s.o + w * s.w + head * s.h; }
};

// Workgroup -> chunk m of a chain: the heads (H of them) of a chunk follow one another on one die (workgroups go to the eight dies in turn), since rows of
// neighbouring heads share lines of memory, which a die's cache holds.  false: there is none.
// (indexes in 32 bits, delta_run sees to it: divisions in 64 were a fifth of a wavefront's instructions in these kernels)
__device__ __forceinline__ bool chunk_of(const DeltaArgs& p, int H, int& chain, int& m) {
    const unsigned id = (unsigned)p.first + blockIdx.x, turn = id >> 3, turns = turn / (unsigned)H;
    const unsigned place = turns * 8 + (id & 7), row = place / (unsigned)p.NC;   // (batch element, chunk)
    m = (int)(place - row * (unsigned)p.NC);
    chain = (int)(row * H + (turn - turns * H));
    return row < (unsigned)(p.O * p.W);
}

// A chunk of a tensor's rows, columns [col, col + R), on its way to LDS: `load` makes the loads, all without a condition where rows lie in pieces of
// 8 (what is not there is read from row 0 and dropped), so that they are under way together with others; `put` leaves planes, 0 behind
// the chain's end and behind the row's end d.  By NT threads, this one `thread` of them.
template <typename T, int NP, int R, int NT = 256>
struct Staged {
    static constexpr int ALL = kDeltaChunk * (R / 8), N = (ALL + NT - 1) / NT, QUADS = sizeof(T) / 2;
    // (as they come: values taken apart here would be waited for here)
    f32x4 v[N][QUADS];
    bool on[N];
    __device__ __forceinline__ void load(const T* base, long long st, const DeltaArgs& p, const DeltaChain& c, int first, int col, int d, bool vec,
                                         int thread = threadIdx.x) {
        int at[N];
        const T* q[N];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int e = thread + n * NT;
            const int i = first + e / (R / 8);
            at[n] = col + e % (R / 8) * 8;
            on[n] = i < c.len && at[n] < d && e < ALL;
            q[n] = base + (on[n] ? (long long)c.step(p, i) * st + at[n] : 0);
        }
        if (vec) {
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int m = 0; m < QUADS; ++m) v[n][m] = reinterpret_cast<const f32x4*>(q[n])[m];
        } else {
#pragma unroll
            for (int n = 0; n < N; ++n) {
                T one[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) one[j] = on[n] && at[n] + j < d ? q[n][j] : from_f32<T>(0.f);
                __builtin_memcpy(v[n], one, sizeof one);
            }
        }
    }
    __device__ __forceinline__ void put(bf16_t* to, int thread = threadIdx.x) const {
        typedef Rows<NP, kDeltaChunk, R> L;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int e = thread + n * NT;
            if (ALL % NT && e >= ALL) continue;
            T one[8];
            __builtin_memcpy(one, v[n], sizeof one);
            Frag<NP> f = planes_of<T, NP>(one);
#pragma unroll
            for (int m = 0; m < NP; ++m) {
                if (!on[n]) f.p[m] = bf16x8{};
                *reinterpret_cast<bf16x8*>(to + m * L::kPlane + e / (R / 8) * L::kStride + e % (R / 8) * 8) = f.p[m];
            }
        }
    }
};

// A plain run of 16-byte pieces from memory to LDS, by NT threads.
template <int BYTES, int NT = 256>
struct Run {
    static constexpr int N = (BYTES / 16 + NT - 1) / NT;
    f32x4 v[N];
    __device__ __forceinline__ void load(const void* from) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int e = threadIdx.x + n * NT;
            v[n] = load_at<f32x4>(from, (e < BYTES / 16 ? e : 0) * 16);
        }
    }
    __device__ __forceinline__ void put(void* to) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int e = threadIdx.x + n * NT;
            if (e < BYTES / 16) *reinterpret_cast<f32x4*>((char*)to + e * 16) = v[n];
        }
    }
};

// The gates of a chunk.  c_i, the sum of the log decays (base 2) up to step i, is summed in 64 bits and kept as two floats, so that differences of
// far sums lose nothing; log decays below -10000 count as that: e^-10000 is 0 in 32 bits, and differences behind it stay exact where a
// mask's lowest value, summed, had swallowed them.  The forward's first launch makes them, the others read them.
struct DeltaGates {
    float hi[kDeltaChunk], lo[kDeltaChunk], beta[kDeltaChunk], D[kDeltaChunk], E[kDeltaChunk];   // D = e^c, E = e^(c_end - c)
    float slope[kDeltaChunk], bslope[kDeltaChunk];   // of the log decay by g, of beta by b
};

__device__ __forceinline__ float gate_value(const void* base, long long at, int f32, int type) {
    if (f32 || type == kF32) return ((const float*)base)[at];
    return type == kF16 ? to_f32(((const f16_t*)base)[at]) : to_f32(((const bf16_t*)base)[at]);
}

// -> log decay and its slope
__device__ __forceinline__ void log_decay(float g, int logits, float& la, float& slope) {
    la = g, slope = 1.f;
    if (logits) {
        const float e = expf(-fabsf(g));
        la = (g < 0.f ? g : 0.f) - log1pf(e);
        slope = (g < 0.f ? 1.f : e) / (1.f + e);   // sigmoid(-g)
        if (g != g) la = slope = g;
    }
    if (la < -104.f) slope = 0.f;   // e^la is 0 in 32 bits, and so is the gradient, which the backward sums of terms that cancel
    if (la < -1e4f) la = -1e4f;
}
__device__ __forceinline__ void write_strength(float b, int logits, float& beta, float& slope) {
    beta = b, slope = 1.f;
    if (logits) {
        const float e = expf(-fabsf(b)), r = 1.f / (1.f + e);
        beta = (b < 0.f ? e : 1.f) * r;
        slope = e * r * r;
        if (b != b) beta = slope = b;
    }
}

// Sums over a wavefront's lanes up to each, in 64 bits: moves within rows of 16 lanes and from row to row, no exchange through LDS.
template <int CTRL, int ROWS>
__device__ __forceinline__ double lanes_before(double v) {
    const unsigned long long bits = __builtin_bit_cast(unsigned long long, v);
    const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)bits, CTRL, ROWS, 0xf, false);
    const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(bits >> 32), CTRL, ROWS, 0xf, false);
    return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);   // (0 where there is no such lane)
}
__device__ __forceinline__ double sums_up_to(double v) {
    v += lanes_before<0x111, 0xf>(v);   // 1, 2, 4 and 8 lanes before
    v += lanes_before<0x112, 0xf>(v);
    v += lanes_before<0x114, 0xf>(v);
    v += lanes_before<0x118, 0xf>(v);
    v += lanes_before<0x142, 0xa>(v);   // the last lane of row 0 to row 1, of row 2 to row 3
    v += lanes_before<0x143, 0xc>(v);   // of row 1 to rows 2 and 3
    return v;
}

// The same in two steps, a load and what its bits mean.
__device__ __forceinline__ unsigned gate_bits(const void* base, long long at, bool wide) {
    return wide ? ((const unsigned*)base)[at] : ((const unsigned short*)base)[at];
}
__device__ __forceinline__ float gate_of(unsigned bits, bool wide, int type) {
    if (wide) return __builtin_bit_cast(float, bits);
    return type == kF16 ? to_f32(__builtin_bit_cast(f16_t, (unsigned short)bits)) : to_f32(__builtin_bit_cast(bf16_t, (unsigned short)bits));
}

// Made by the first wavefront, in two steps (loads ahead of others; the rest), into LDS and memory; the caller's barrier follows.
struct GateMaker {
    unsigned gbits, bbits;
    bool on;
    __device__ __forceinline__ void load(const DeltaArgs& p, const DeltaChain& c, int first, int type) {
        const int i = first + (threadIdx.x & 63);
        on = i < c.len;
        const long long t = on ? c.step(p, i) : 0;
        const bool wide = p.gates_f32 || type == kF32;
        gbits = gate_bits(p.g, c.at(p.gs, c.hv) + t * p.gs.t, wide);
        bbits = gate_bits(p.b, c.at(p.bs, c.hv) + t * p.bs.t, wide);
    }
    __device__ __forceinline__ void make(DeltaGates& s, DeltaGates* to, const DeltaArgs& p, int type) {
        const int lane = threadIdx.x & 63;
        const bool wide = p.gates_f32 || type == kF32;
        const float g = gate_of(gbits, wide, type), b = gate_of(bbits, wide, type);
        float la, slope, beta, bslope;
        log_decay(g, p.logits, la, slope);
        write_strength(b, p.logits, beta, bslope);
        if (!on) la = slope = beta = bslope = 0.f;
        const double sum = sums_up_to(la * 1.4426950408889634), end = __shfl(sum, 63);
        const float hi = (float)sum, lo = (float)(sum - (double)hi), D = __builtin_amdgcn_exp2f(hi), E = __builtin_amdgcn_exp2f((float)(end - sum));
        s.hi[lane] = to->hi[lane] = hi, s.lo[lane] = to->lo[lane] = lo, s.beta[lane] = to->beta[lane] = beta;
        s.D[lane] = to->D[lane] = D, s.E[lane] = to->E[lane] = E;
        s.slope[lane] = to->slope[lane] = slope, s.bslope[lane] = to->bslope[lane] = bslope;
    }
};

// e^(c_i - c_j) of a tile: this lane's step and four others of it, which is i and which j: rows: this lane's is i.  Above the diagonal (i < j) it may
// be infinite: the caller selects.
struct TileDecay {
    f32x4 G, beta;   // beta of the rows i
    __device__ __forceinline__ TileDecay(const DeltaGates& s, int mine, int others, bool rows) {
        const f32x4 hi = *reinterpret_cast<const f32x4*>(s.hi + others), lo = *reinterpret_cast<const f32x4*>(s.lo + others);
        beta = *reinterpret_cast<const f32x4*>(s.beta + others);
        const float h = s.hi[mine], l = s.lo[mine], b = s.beta[mine], sign = rows ? 1.f : -1.f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            G[r] = __builtin_amdgcn_exp2f(sign * ((h - hi[r]) + (l - lo[r])));
            beta[r] = rows ? b : beta[r];
        }
    }
};

// (I + A)^-1 of a chunk, A strictly lower, as blocks of 16 x 16 for a substitution by blocks: -A_ba below the diagonal, the inverses of the
// diagonal's blocks on it.  Block (b, a) is number b (b + 1) / 2 + a.  Lane = row, values = columns, an operand for products with
// solutions by their rows; turned, lane = column, values = rows: the same for the transposed system.
template <int NP>
struct Blocks {
    static constexpr int kValues = 10 * NP * 64 * 4;
    static __device__ __forceinline__ int at(int b, int a) { return b * (b + 1) / 2 + a; }
    static __device__ __forceinline__ void put(bf16_t* base, int block, const Half<NP>& h, int lane) {
#pragma unroll
        for (int p = 0; p < NP; ++p) *reinterpret_cast<bf16x4*>(base + ((block * NP + p) * 64 + lane) * 4) = h.p[p];
    }
    static __device__ __forceinline__ Half<NP> get(const bf16_t* base, int block, int lane) {
        Half<NP> h;
#pragma unroll
        for (int p = 0; p < NP; ++p) h.p[p] = *reinterpret_cast<const bf16x4*>(base + ((block * NP + p) * 64 + lane) * 4);
        return h;
    }
};

// The inverse T of a block I + A, strictly lower A with lane = row, values = columns, as it is: row i of T from T (I + A) = I,
// t_j = [i = j] - sum over m > j of t_m A_mj, from the last column.  A lane has a row; A's elements come to all lanes as scalars.
__device__ __forceinline__ f32x4 invert_block(f32x4 A, int lane) {
    const int me = lane & 15;
    float t[16];
#pragma unroll
    for (int j = 15; j >= 0; --j) {
        float s = j == me ? 1.f : 0.f;
        // (the latest of t last: it is what there is to wait for)
#pragma unroll
        for (int m = 15; m > j; --m) {
            const float row = A[j & 3];   // (a bit cast of an element would take the first one)
            s = __builtin_fmaf(-t[m], __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, row), (j >> 2) * 16 + m)), s);
        }
        t[j] = s;
    }
    f32x4 v;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int g = lane >> 4;
        v[r] = g == 0 ? t[r] : g == 1 ? t[4 + r] : g == 2 ? t[8 + r] : t[12 + r];
    }
    return v;
}

// What is not finite.  A chunk's products run over blocks of steps, with zeros where a step has no part in another, and 0 times NaN is NaN: a bad row
// would reach the steps before it.  Where a result says that there may be one (rare: one comparison), the product is made again without the rows
// from a column's first bad one on, and from that step on the column is NaN, as its state is from there on.  (The limit: rounded to bf16 it is infinite.)
__device__ __forceinline__ bool is_bad(float v) { return !(__builtin_fabsf(v) < 0x1.ffp127f); }
__device__ __forceinline__ int first_of_groups(int n) {   // the least over the four lane groups
    int m = __shfl_xor(n, 16);
    n = m < n ? m : n;
    m = __shfl_xor(n, 32);
    return m < n ? m : n;
}

// A block's inverse with such rows (a lane has a row): those before them have no part in them.
__device__ __forceinline__ f32x4 invert_rows(f32x4 A, int lane) {
    const unsigned long long b = __ballot(is_bad(A[0]) || is_bad(A[1]) || is_bad(A[2]) || is_bad(A[3]));
    const unsigned rows = (unsigned)(b | b >> 16 | b >> 32 | b >> 48) & 0xffffu;
    const bool behind = rows && (lane & 15) >= __builtin_ctz(rows | 0x10000u);
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f}, nan = zero + __builtin_nanf("");
    const f32x4 t = invert_block(behind ? zero : A, lane);
    return behind ? nan : t;
}

// Solutions X of (I + A) X = R f by blocks of rows: lane = column, values = rows, each with a factor of its own.  A solved block goes at once into the rows
// behind it.
template <int NP>
__device__ __forceinline__ void solve_fore(const bf16_t* blocks, const f32x4 (&R)[4], const f32x4 (&f)[4], f32x4 (&x)[4], int lane) {
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int b = 1; b < 4; ++b) x[b] = R[b] * f[b];
#pragma unroll
    for (int a = 0; a < 4; ++a) {
        x[a] = mma(Blocks<NP>::get(blocks, Blocks<NP>::at(a, a), lane), a ? split<NP>(x[a]) : split_product<NP>(R[0], f[0]), zero);
        const Half<NP> s = split<NP>(x[a]);
#pragma unroll
        for (int b = a + 1; b < 4; ++b) x[b] = mma(Blocks<NP>::get(blocks, Blocks<NP>::at(b, a), lane), s, x[b]);
    }
}
// The same where rows are bad, of R f or of the system.  (After solve_fore a column's row 48 is NaN where a bad row has reached others.)
template <int NP>
__device__ __forceinline__ void solve_fore_until(const bf16_t* blocks, f32x4 (&R)[4], f32x4 (&f)[4], f32x4 (&x)[4], int lane) {
    const int g4 = 4 * (lane >> 4);
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    int first = kDeltaChunk;
    auto look = [&](int a) {
        int n = kDeltaChunk;
#pragma unroll
        for (int r = 3; r >= 0; --r) n = is_bad(x[a][r]) ? 16 * a + g4 + r : n;
        n = first_of_groups(n);
        first = n < first ? n : first;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const bool before = 16 * a + g4 + r < first;
            x[a][r] = before ? x[a][r] : 0.f, R[a][r] = before ? R[a][r] : 0.f, f[a][r] = before ? f[a][r] : 0.f;
        }
    };
#pragma unroll
    for (int b = 0; b < 4; ++b) x[b] = R[b] * f[b];
#pragma unroll
    for (int a = 0; a < 4; ++a) {
        look(a);
        x[a] = mma(Blocks<NP>::get(blocks, Blocks<NP>::at(a, a), lane), a ? split<NP>(x[a]) : split_product<NP>(R[0], f[0]), zero);
        look(a);
        const Half<NP> s = split<NP>(x[a]);
#pragma unroll
        for (int b = a + 1; b < 4; ++b) x[b] = mma(Blocks<NP>::get(blocks, Blocks<NP>::at(b, a), lane), s, x[b]);
    }
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int r = 0; r < 4; ++r) x[a][r] = 16 * a + g4 + r < first ? x[a][r] : __builtin_nanf("");
}
// of (I + A)^T X = R, from the last block.
template <int NP>
__device__ __forceinline__ void solve_back(const bf16_t* blocks, f32x4 (&x)[4], int lane) {
#pragma unroll
    for (int b = 3; b >= 0; --b) {
        const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
        x[b] = mma(Blocks<NP>::get(blocks, Blocks<NP>::at(b, b), lane), split<NP>(x[b]), zero);
        const Half<NP> s = split<NP>(x[b]);
#pragma unroll
        for (int a = b - 1; a >= 0; --a) x[a] = mma(Blocks<NP>::get(blocks, Blocks<NP>::at(b, a), lane), s, x[a]);
    }
}

// Fragments in memory: [fragment][plane][lane][8].
template <int NP>
__device__ __forceinline__ void store_frag(bf16_t* base, int fragment, const Frag<NP>& f, int lane) {
#pragma unroll
    for (int p = 0; p < NP; ++p) store_at(base + (fragment * NP + p) * 512, lane * 16, f.p[p]);
}
template <int NP>
__device__ __forceinline__ Frag<NP> load_frag(const bf16_t* base, int fragment, int lane) {
    Frag<NP> f;
#pragma unroll
    for (int p = 0; p < NP; ++p) f.p[p] = load_at<bf16x8>(base + (fragment * NP + p) * 512, lane * 16);
    return f;
}
// A tile of what lies as fragments with lane = column of v and values = rows (states, U), with lane = row and values = columns: rows of tile `t` of 16,
// two tiles of columns, whose fragments are `stride` apart.
template <int NP>
__device__ __forceinline__ Frag<NP> load_turned(const bf16_t* base, int fragment, int stride, int half, bf16x4 unit, int lane) {
    Half<NP> a, b;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        a.p[p] = load_at<bf16x4>(base + (fragment * NP + p) * 512 + 4 * half, lane * 16);
        b.p[p] = load_at<bf16x4>(base + ((fragment + stride) * NP + p) * 512 + 4 * half, lane * 16);
    }
#pragma unroll
    for (int p = 0; p < NP; ++p) a.p[p] = turned(a.p[p], unit), b.p[p] = turned(b.p[p], unit);
    return join(a, b);
}
// one of the two tiles of a fragment
template <int NP>
__device__ __forceinline__ void store_half(bf16_t* base, int fragment, int half, const Half<NP>& h, int lane) {
#pragma unroll
    for (int p = 0; p < NP; ++p)
        store_at(base + (fragment * NP + p) * 512 + 4 * half, lane * 16, h.p[p]);
}

// Four neighbouring values of a row of d to memory.
template <typename T>
__device__ __forceinline__ void store_four(T* row, int at, int d, f32x4 v, bool vec) {
    if (vec) {
        if (at < d) {
            const float f[4] = {v[0], v[1], v[2], v[3]};
            store_f32<T, 4>(row + at, f);
        }
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (at + r < d) row[at + r] = from_f32<T>(v[r]);
    }
}

// The sum over the four lane groups, in all of them.
__device__ __forceinline__ float group_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// Sizes of what lies between the kernels, in elements of a chunk; of a segment's map.
struct DeltaSizes {
    long long w, state, u, cols, c0, map, shift, blocks;
    __host__ __device__ DeltaSizes(int DK, int dvp, int made, int chain)
        : w(kDeltaChunk * (long long)DK), state((long long)DK * dvp * made), u((long long)kDeltaChunk * dvp * made),
          cols((long long)kDeltaChunk * dvp), c0((long long)DK * dvp), map((long long)DK * DK * chain), shift((long long)DK * dvp),
          blocks(10 * made * 256) {}
};

}  // namespace pdw
