// The gated delta rule's chains, forward and backward: the only part with an order in time.  A state's columns X pass through the chunks,
//
//   forward    U = Ub - W X,          leaves X (the state before the chunk) and U,       X' = e^c_end X + K^T E U
//   backward   Y = E K X, dU += Y,    leaves X (the gradient of the state behind it),    X' = e^c_end X + C - W^T Y       (from the last chunk)
//
// two products a chunk: A X, and B of the first one's result.  A wavefront carries 16 columns in registers; results of one product are
// operands of the next as they are.  A and B come as fragments from memory and are the same for all columns of a chain, so other wavefronts of
// the workgroup fetch them, several chunks ahead in registers, and put them into LDS: A's place is filled while B is in use and the other way round, two
// barriers a chunk.  What bounds it: latencies, of the products and of the exchange between the wavefronts, one chunk after another.
//
// Where there are too few chains to fill the chip, the chunks are cut into segments.  Through a segment X goes to M X + N, and the same kernel
// (MAPS) finds both: N from X = 0, and M as what becomes of the unit matrix' columns without what the chunks add.  delta_join_k takes the states
// through the maps, from segment to segment, and the second launch begins each segment with its own.
#pragma once
#include "delta_common.h"

namespace pdw {

// A state's 16 columns: X[d] has rows 16 d + 4 g + r, lane = column.  From and to the user's [dk][dv].
template <int DK>
__device__ __forceinline__ void load_state(f32x4 (&x)[DK / 16], const float* s, int dk, int dv, int at, int lane) {
#pragma unroll
    for (int d = 0; d < DK / 16; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 16 * d + 4 * (lane >> 4) + r;
            x[d][r] = s && row < dk && at < dv ? s[row * (long long)dv + at] : 0.f;
        }
}
template <int DK>
__device__ __forceinline__ void store_state(float* s, const f32x4 (&x)[DK / 16], int dk, int dv, int at, int lane) {
    if (!s) return;
#pragma unroll
    for (int d = 0; d < DK / 16; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 16 * d + 4 * (lane >> 4) + r;
            if (row < dk && at < dv) s[row * (long long)dv + at] = x[d][r];
        }
}
template <typename T, bool BACK, int CP>
struct ChainPlanes {
    static constexpr int kRaw = DeltaPlanes<T>::kRaw;
    static constexpr int kA = BACK ? kRaw : CP, kB = BACK ? CP : kRaw;   // planes of A and of B
};
template <typename T, int DK, bool BACK, int CP>
constexpr int delta_chain_lds() {
    typedef ChainPlanes<T, BACK, CP> P;
    return kDeltaChunk * DK * (P::kA + P::kB) * 2;
}

// What a workgroup's index stands for: segments of a chain's column parts; the parts of a chain, which read the same operands, on one die (workgroups go to
// the eight dies in turn).
__device__ __forceinline__ bool chain_part(const DeltaArgs& p, int parts, int segments, int& chain, int& part, int& segment) {
    const long long id = p.first + blockIdx.x;
    long long turn = id >> 3;
    part = (int)(turn % parts), turn /= parts;
    segment = (int)(turn % segments);
    const long long n = turn / segments * 8 + (id & 7);
    chain = (int)n;
    return n < p.chains;
}

// Wavefronts that carry columns, at least (and as many fetch): with 64 channels fewer had no registers for what they fetch.
template <int DK>
constexpr int delta_least_waves() {
    return DK >= 64 ? 4 : 2;
}

// Chunks that are under way: a chunk is done in less time than its operands take from memory; as many as there are registers for.
template <int DK, bool BACK>
constexpr int delta_ahead() {
    return DK == 32 ? 4 : DK == 64 ? 3 : 2;
}

// Half of the workgroup's wavefronts carry columns, half fetch.
template <typename T, int DK, bool BACK, int CP, bool MAPS>
__global__ __launch_bounds__(512) void delta_chain_k(DeltaArgs p) {
    typedef ChainPlanes<T, BACK, CP> P;
    constexpr int RAW = P::kRaw, MADE = DeltaPlanes<T>::kMade, ND = DK / 16, NA = 4 * (DK / 32) * P::kA, NB = ND * 2 * P::kB;   // fragments' planes
    constexpr int kLeast = delta_least_waves<DK>(), AHEAD = delta_ahead<DK, BACK>(), ROWS = ND < 4 ? ND : 4;
    extern __shared__ __align__(16) unsigned char lds[];
    bf16_t *la = (bf16_t*)lds, *lb = la + NA * 512;
    const int lane = threadIdx.x & 63, waves = blockDim.x >> 7, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g4 = 4 * (lane >> 4), colv = p.dvp / 16, cols = MAPS ? colv + ND : colv;
    int chain, part, segment;
    if (!chain_part(p, (cols + waves - 1) / waves, MAPS ? p.segments - 1 : p.segments, chain, part, segment)) return;
    const DeltaSizes z(DK, p.dvp, RAW, MADE, CP);
    // chunks in the chain's order: n of them from `from`, each `by` behind the last
    const long long place = segment * p.seg, n = p.NC - place < p.seg ? p.NC - place : p.seg;
    const long long by = BACK ? -1 : 1, from = chain * p.NC + (BACK ? p.NC - 1 - place : place);

    if (wave >= waves) {
        const int w = wave - waves;
        const bf16_t* ga = BACK ? p.ka : p.wp;
        const bf16_t* gb = BACK ? p.wp : p.kt;
        const long long sa = kDeltaChunk * DK * P::kA, sb = kDeltaChunk * DK * P::kB;
        constexpr int RA = (NA + kLeast - 1) / kLeast, RB = (NB + kLeast - 1) / kLeast;
        bf16x8 a[AHEAD][RA], b[AHEAD][RB];
        auto fetch = [&](bf16x8* r, const bf16_t* base, int count, int most) {
#pragma unroll
            for (int i = 0; i < most; ++i) {
                const int f = i * waves + w;
                if (f < count) r[i] = load_at<bf16x8>(base + f * 512, lane * 16);
            }
        };
        auto put = [&](const bf16x8* r, bf16_t* base, int count, int most) {
#pragma unroll
            for (int i = 0; i < most; ++i) {
                const int f = i * waves + w;
                if (f < count) store_at(base + f * 512, lane * 16, r[i]);
            }
        };
        auto fetch_a = [&](int j, long long m) {
            if (m < n) fetch(a[j], ga + (from + m * by) * sa, NA, RA);
        };
        auto fetch_b = [&](int j, long long m) {
            if (m < n) fetch(b[j], gb + (from + m * by) * sb, NB, RB);
        };
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) fetch_a(j, j), fetch_b(j, j);
        put(a[0], la, NA, RA);
        fetch_a(0, AHEAD);
        __syncthreads();
        for (long long m0 = 0; m0 < n; m0 += AHEAD) {
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const long long m = m0 + j;
                if (m >= n) break;
                put(b[j], lb, NB, RB);
                fetch_b(j, m + AHEAD);
                __syncthreads();
                constexpr int last = AHEAD - 1;
                const int k = j == last ? 0 : j + 1;
                if (m + 1 < n) put(a[k], la, NA, RA);
                fetch_a(k, m + 1 + AHEAD);
                __syncthreads();
            }
        }
        return;
    }

    const int cv = part * waves + wave;
    const bool on = cv < cols, unit_cols = MAPS && cv >= colv;   // (a wavefront without columns of its own goes along)
    const bf16x4 unit = unit_half(lane);
    const int at = 16 * cv + (lane & 15);
    const long long state = (long long)chain * p.dk * p.dv;
    f32x4 x[ND];
    if constexpr (MAPS) {
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) x[d][r] = 16 * d + g4 + r == at - 16 * colv ? 1.f : 0.f;
    } else {
        const float* h = BACK ? p.glast : p.h0;
        if (segment == 0) {
            load_state<DK>(x, h ? h + state : nullptr, p.dk, p.dv, on ? at : p.dv, lane);
        } else {
            const float* from_maps = p.shifts + (chain * (long long)(p.segments - 1) + segment - 1) * z.shift + cv * (DK * 16);
#pragma unroll
            for (int d = 0; d < ND; ++d) x[d] = on ? load_at<f32x4>(from_maps + d * 256, lane * 16) : f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }

    // what a chunk brings to these columns
    struct Chunk {
        f32x4 y0[4], E[4];
        float end;
    };
    auto fetch = [&](Chunk& c, long long id) {
        const float *y0 = (BACK ? p.du : p.ub) + id * z.cols + cv * 1024;
        const DeltaGates* s = p.gates + id;
        const bool own = on && !unit_cols;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            c.y0[b] = own && !(BACK && MAPS) ? load_at<f32x4>(y0 + b * 256, lane * 16) : f32x4{0.f, 0.f, 0.f, 0.f};
            c.E[b] = load_at<f32x4>(s->E + 16 * b, g4 * 4);
        }
        c.end = s->D[kDeltaChunk - 1];
    };
    Chunk chunks[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
        if (j < n) fetch(chunks[j], from + j * by);
    __syncthreads();
    for (long long m0 = 0; m0 < n; m0 += AHEAD)
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
        const long long m = m0 + j, id = from + m * by;
        if (m >= n) break;
        const Chunk& c = chunks[j];
        f32x4 c0[BACK ? ND : 1];
        if constexpr (BACK) {
#pragma unroll
            for (int d = 0; d < ND; ++d)
                c0[d] = on && !unit_cols ? load_at<f32x4>(p.c0 + id * z.c0 + cv * (DK * 16) + d * 256, lane * 16) : f32x4{0.f, 0.f, 0.f, 0.f};
        }
        Frag<CP> xs[DK / 32];
#pragma unroll
        for (int d = 0; d < DK / 32; ++d) xs[d] = join(split<CP>(x[2 * d]), split<CP>(x[2 * d + 1]));
        f32x4 y[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) y[b] = BACK ? f32x4{0.f, 0.f, 0.f, 0.f} : c.y0[b];
#pragma unroll
        for (int d = 0; d < DK / 32; ++d) {
            Frag<P::kA> a[4];
#pragma unroll
            for (int b = 0; b < 4; ++b) a[b] = load_frag<P::kA>(la, b * (DK / 32) + d, lane);
            mma_rows(a, xs[d], y);
        }
        if constexpr (!MAPS) {
            if (on) {
                bf16_t* to = (BACK ? p.ds1 : p.s0) + id * z.state;
#pragma unroll
                for (int d = 0; d < DK / 32; ++d) store_frag(to, cv * (DK / 32) + d, planes<MADE>(xs[d]), lane);
            }
        }
        __syncthreads();
        Half<CP> e[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) e[b] = split<CP>(y[b] * c.E[b]);
        const Frag<CP> e0 = join(e[0], e[1]), e1 = join(e[2], e[3]);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            x[d] = x[d] * c.end;
            if constexpr (BACK) x[d] += c0[d];
        }
#pragma unroll
        for (int d0 = 0; d0 < ND; d0 += ROWS) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                Frag<P::kB> a[ROWS];
                f32x4 t[ROWS];
#pragma unroll
                for (int d = 0; d < ROWS; ++d) a[d] = load_frag<P::kB>(lb, 2 * (d0 + d) + h, lane), t[d] = x[d0 + d];
                mma_rows(a, h ? e1 : e0, t);
#pragma unroll
                for (int d = 0; d < ROWS; ++d) x[d0 + d] = t[d];
            }
        }
        if constexpr (!MAPS) {
            if (on) {
                if constexpr (BACK) {
#pragma unroll
                    for (int b = 0; b < 4; ++b) store_at(p.du + id * z.cols + cv * 1024 + b * 256, lane * 16, c.y0[b] + y[b] * c.E[b]);
                } else {
                    bf16_t* to = p.u + id * z.u;
                    store_frag(to, cv * 2, join(split<MADE>(y[0]), split<MADE>(y[1])), lane);
                    store_frag(to, cv * 2 + 1, join(split<MADE>(y[2]), split<MADE>(y[3])), lane);
                }
            }
        }
        if (m + AHEAD < n) fetch(chunks[j], id + AHEAD * by);
        __syncthreads();
    }
    if constexpr (MAPS) {
        const long long id = chain * (long long)(p.segments - 1) + segment;
        if (!on) return;
        if (!unit_cols) {
#pragma unroll
            for (int d = 0; d < ND; ++d) store_at(p.shifts + id * z.shift + cv * (DK * 16) + d * 256, lane * 16, x[d]);
        } else {
            // rows of M as a first operand: lane = row, values = columns
            const int ct = cv - colv;
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                Half<CP> h = split<CP>(x[d]);
#pragma unroll
                for (int q = 0; q < CP; ++q) h.p[q] = turned(h.p[q], unit);
                store_half(p.maps + id * z.map, d * (DK / 32) + ct / 2, ct & 1, h, lane);
            }
        }
    } else if (segment == p.segments - 1 && on) {
        float* to = BACK ? p.gh0 : p.last;
        store_state<DK>(to ? to + state : nullptr, x, p.dk, p.dv, at, lane);
    }
}

// The state before every segment but the first, in the place of its predecessor's shift N: X = M X + N from segment to segment.  A workgroup has 16 columns
// of a chain, a wavefront 16 rows of them: its rows of M are under way while the last segment's product is made, X goes round through LDS.
template <typename T, int DK, bool BACK, int CP>
__global__ __launch_bounds__(DK * 4) void delta_join_k(DeltaArgs p) {
    constexpr int NK = DK / 32;
    __shared__ __align__(16) bf16_t lx[2][NK * CP * 512];
    const int lane = threadIdx.x & 63, d = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), colv = p.dvp / 16;
    const long long id = p.first + blockIdx.x;
    const int chain = (int)(id / colv), cv = (int)(id - (long long)chain * colv);
    const DeltaSizes z(DK, p.dvp, 1, 1, CP);
    const float* h = BACK ? p.glast : p.h0;
    const int at = 16 * cv + (lane & 15);
    f32x4 x;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int row = 16 * d + 4 * (lane >> 4) + r;
        x[r] = h && row < p.dk && at < p.dv ? h[((long long)chain * p.dk + row) * p.dv + at] : 0.f;
    }
    const bf16_t* maps = p.maps + chain * (long long)(p.segments - 1) * z.map;
    float* shifts = p.shifts + chain * (long long)(p.segments - 1) * z.shift + cv * (DK * 16) + d * 256;
    Frag<CP> m[NK];
    f32x4 n;
    auto fetch = [&](int s) {
#pragma unroll
        for (int k = 0; k < NK; ++k) m[k] = load_frag<CP>(maps + s * z.map, d * NK + k, lane);
        n = load_at<f32x4>(shifts + s * z.shift, lane * 16);
    };
    fetch(0);
    for (int s = 0; s + 1 < p.segments; ++s) {
        bf16_t* l = lx[s & 1];
        store_half(l, d / 2, d & 1, split<CP>(x), lane);
        __syncthreads();
        f32x4 t[NK];
#pragma unroll
        for (int k = 0; k < NK; ++k) t[k] = mma(m[k], load_frag<CP>(l, k, lane), k ? f32x4{0.f, 0.f, 0.f, 0.f} : n);
        x = t[0];
#pragma unroll
        for (int k = 1; k < NK; ++k) x += t[k];
        float* to = shifts + s * z.shift;
        if (s + 2 < p.segments) fetch(s + 1);
        store_at(to, lane * 16, x);
    }
}

}  // namespace pdw
