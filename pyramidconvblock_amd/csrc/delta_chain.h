// The gated delta rule's chains, forward and backward: the only part with an order in time.  A state's columns X pass through the chunks,
//
//   forward    U = Ub - W X,    leaves X (the state before the chunk) and U,      X' = e^c_end X + K^T E U
//   backward   Y = E K X,       leaves X (the gradient of the state behind it),   X' = e^c_end X + C - W^T Y       (from the last chunk)
//
// two products a chunk, with W (from memory in fp32: fewer bytes than its planes) and K (from the tensor).  A wavefront carries 16 columns in registers;
// results of one product are operands of the next as they are.  W and K are the same for all columns of a chain, so other wavefronts of the workgroup
// fetch them, several chunks ahead in registers, and put them into LDS: one's place is filled while the other is in use, a barrier
// a chunk, or two where LDS has no room for both.  What bounds it: with many chains memory (240 segments of 13 chunks at 64 channels
// in fp16: 232 MB in 43 us), with few the latencies of splits, products and the exchange between the wavefronts, one chunk after another (1.6 us a chunk at 32
// channels, 2.7 at 64, 3.5 at 128).
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
// W's planes as its tiles come (lane = channel of k, values = steps), [plane][tile of channels][tile of steps][lane][4], and K's rows.
template <typename T, int DK, int CP>
constexpr int delta_chain_values() {
    return kDeltaChunk * DK * CP + Rows<DeltaPlanes<T>::kRaw, kDeltaChunk, DK>::kValues;
}
// Twice where there is room: a chunk's operands are put while the last one's are in use, with one barrier a chunk (77 us for 80 with two at 128 chains of 49
// chunks of 32 channels in bf16, 110 for 116 at 12 of 256 of 64 in fp16); fp16's and fp32's 128 channels have none.
template <typename T, int DK, int CP>
constexpr bool delta_chain_twice() {
    return delta_chain_values<T, DK, CP>() * 4 <= 160 * 1024;
}
template <typename T, int DK, int CP>
constexpr int delta_chain_lds() {
    return delta_chain_values<T, DK, CP>() * (delta_chain_twice<T, DK, CP>() ? 4 : 2);
}

// What a workgroup's index stands for: the column parts of a chain's segments; the parts of a segment, which read the same operands, on one die (workgroups
// go to the eight dies in turn), and segments on one after another (with a chain to a die, twelve chains leave half of the dies
// half idle: 99 us for 71, 20 segments each at 64 channels).
__device__ __forceinline__ bool chain_part(const DeltaArgs& p, int parts, int segments, int& chain, int& part, int& segment) {
    const unsigned id = (unsigned)p.first + blockIdx.x, turn = id >> 3, turns = turn / (unsigned)parts, n = turns * 8 + (id & 7);
    part = (int)(turn - turns * parts);
    chain = (int)(n / (unsigned)segments);
    segment = (int)(n - (unsigned)chain * segments);
    return chain < p.chains;
}

// Wavefronts that carry columns, at least (and as many fetch): with 64 channels fewer had no registers for what they fetch.
template <int DK>
constexpr int delta_least_waves() {
    return DK >= 64 ? 4 : 2;
}

// Chunks that are under way: a chunk is done in less time than its operands take from memory; as many as there are registers for.
template <int DK>
constexpr int delta_ahead() {
    return DK == 32 ? 4 : DK == 64 ? 3 : 2;
}

// What is fetched of a chunk by NT threads of NT / 64 wavefronts: W's tiles (in fp32, split on the way) and K's rows.
template <typename T, int DK, int CP, int NT>
struct ChainFetch {
    static constexpr int RAW = DeltaPlanes<T>::kRaw, N = DK / 16 * 4 * 64 / NT;
    f32x4 w[N];
    Staged<T, RAW, DK, NT> k;
    __device__ __forceinline__ void load_w(const DeltaArgs& p, const DeltaSizes& z, long long id, int thread) {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = load_at<f32x4>(p.w + id * z.w, (i * NT + thread) * 16);
    }
    __device__ __forceinline__ void put_w(bf16_t* to, int thread) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const Half<CP> h = split<CP>(w[i]);
#pragma unroll
            for (int q = 0; q < CP; ++q) *reinterpret_cast<bf16x4*>(to + q * (kDeltaChunk * DK) + (i * NT + thread) * 4) = h.p[q];
        }
    }
    __device__ __forceinline__ void load_k(const DeltaArgs& p, const DeltaChain& c, int chunk, int thread) {
        k.load((const T*)p.k + c.at(p.ks, c.hk), p.ks.t, p, c, chunk * kDeltaChunk, 0, p.dk, p.vec & kVecK, thread);
    }
};

template <typename T, int DK, bool BACK, int CP, int NT, int AHEAD>
__device__ __forceinline__ void chain_fetch(const DeltaArgs& p, const DeltaSizes& z, int chain, int chunk, int by, int n, bf16_t* lw, bf16_t* lk,
                                            int thread) {
    const DeltaChain c(p, chain);
    const long long id = (long long)chain * p.NC + chunk;
    ChainFetch<T, DK, CP, NT> f[AHEAD];
    // A is what the first product takes, B the second's: W and K, or (BACK) K and W.  (Behind the last chunk the last once more: loads on a condition would all
    // be waited for where the first of them is, since their number is not known there.)
    auto fetch_a = [&](int j, int m) {
        m = m < n ? m : n - 1;
        if constexpr (BACK) f[j].load_k(p, c, chunk + m * by, thread);
        else f[j].load_w(p, z, id + m * by, thread);
    };
    auto fetch_b = [&](int j, int m) {
        m = m < n ? m : n - 1;
        if constexpr (BACK) f[j].load_w(p, z, id + m * by, thread);
        else f[j].load_k(p, c, chunk + m * by, thread);
    };
    if constexpr (delta_chain_twice<T, DK, CP>()) {
        auto put = [&](int j, int m) {
            const int other = (m & 1) * delta_chain_values<T, DK, CP>();
            f[j].put_w(lw + other, thread), f[j].k.put(lk + other, thread);
        };
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) fetch_a(j, j), fetch_b(j, j);
        put(0, 0);
        fetch_a(0, AHEAD), fetch_b(0, AHEAD);
        __syncthreads();
        for (int m0 = 0; m0 < n; m0 += AHEAD) {
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const int m = m0 + j, k = j == AHEAD - 1 ? 0 : j + 1;
                if (m >= n) break;
                put(k, m + 1);
                fetch_a(k, m + 1 + AHEAD), fetch_b(k, m + 1 + AHEAD);
                __syncthreads();
            }
        }
        return;
    }
    auto put_a = [&](int j) {
        if constexpr (BACK) f[j].k.put(lk, thread);
        else f[j].put_w(lw, thread);
    };
    auto put_b = [&](int j) {
        if constexpr (BACK) f[j].put_w(lw, thread);
        else f[j].k.put(lk, thread);
    };
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) fetch_a(j, j), fetch_b(j, j);
    put_a(0);
    fetch_a(0, AHEAD);
    __syncthreads();
    for (int m0 = 0; m0 < n; m0 += AHEAD) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int m = m0 + j;
            if (m >= n) break;
            put_b(j);
            fetch_b(j, m + AHEAD);
            __syncthreads();
            const int k = j == AHEAD - 1 ? 0 : j + 1;
            put_a(k);
            fetch_a(k, m + 1 + AHEAD);
            __syncthreads();
        }
    }
}

// Half of the workgroup's wavefronts carry columns, half fetch.
template <typename T, int DK, bool BACK, int CP, bool MAPS, int WAVES>
__global__ __launch_bounds__(128 * WAVES) void delta_chain_k(DeltaArgs p) {
    constexpr int RAW = DeltaPlanes<T>::kRaw, MADE = DeltaPlanes<T>::kMade, ND = DK / 16, NK = DK / 32;
    constexpr int AHEAD = delta_ahead<DK>(), ROWS = ND < 4 ? ND : 4, PLANE = kDeltaChunk * DK;
    typedef Rows<RAW, kDeltaChunk, DK> L;
    constexpr bool TWICE = delta_chain_twice<T, DK, CP>();
    extern __shared__ __align__(16) unsigned char lds[];
    bf16_t *lw = (bf16_t*)lds, *lk = lw + CP * PLANE;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g4 = 4 * (lane >> 4), colv = p.dvp / 16, cols = MAPS ? colv + ND : colv;
    int chain, part, segment;
    if (!chain_part(p, (cols + WAVES - 1) / WAVES, MAPS ? p.segments - 1 : p.segments, chain, part, segment)) return;
    const DeltaSizes z(DK, p.dvp, MADE, CP);
    // chunks in the chain's order: n of them from `from`, each `by` behind the last
    const int place = segment * p.seg, n = p.NC - place < p.seg ? p.NC - place : p.seg;
    const int by = BACK ? -1 : 1, chunk = BACK ? p.NC - 1 - place : place;
    const long long from = (long long)chain * p.NC + chunk;

    if (wave >= WAVES)
        return chain_fetch<T, DK, BACK, CP, 64 * WAVES, AHEAD>(p, z, chain, chunk, by, n, lw, lk, threadIdx.x - 64 * WAVES);

    const int cv = part * WAVES + wave;
    if (cv >= cols) {   // without columns: along to the barriers
        __syncthreads();
        for (int m = 0; m < n; ++m) {
            if constexpr (!TWICE) __syncthreads();
            __syncthreads();
        }
        return;
    }
    const bool unit_cols = MAPS && cv >= colv;
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
            load_state<DK>(x, h ? h + state : nullptr, p.dk, p.dv, at, lane);
        } else {
            const float* from_maps = p.shifts + (chain * (long long)(p.segments - 1) + segment - 1) * z.shift + cv * (DK * 16);
#pragma unroll
            for (int d = 0; d < ND; ++d) x[d] = load_at<f32x4>(from_maps + d * 256, lane * 16);
        }
    }

    // what a chunk brings to these columns (to the unit matrix' nothing: it is loaded for another and dropped, as behind the last chunk)
    const int source = unit_cols ? 0 : cv;
    struct Chunk {
        f32x4 y0[BACK ? 1 : 4], E[4];
        float end;
    };
    auto fetch = [&](Chunk& c, int m) {
        const long long id = from + (m < n ? m : n - 1) * by;
        const DeltaGates* s = p.gates + id;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            if constexpr (!BACK) c.y0[b] = load_at<f32x4>(p.ub + id * z.cols + source * 1024 + b * 256, lane * 16);
            c.E[b] = load_at<f32x4>(s->E + 16 * b, g4 * 4);
        }
        c.end = s->D[kDeltaChunk - 1];
    };
    f32x4 c0[BACK ? ND : 1];   // of the next chunk
    auto fetch_c0 = [&](int m) {
        const long long id = from + (m < n ? m : n - 1) * by;
        if constexpr (BACK) {
#pragma unroll
            for (int d = 0; d < ND; ++d) c0[d] = load_at<f32x4>(p.c0 + id * z.c0 + source * (DK * 16) + d * 256, lane * 16);
        }
    };
    Chunk chunks[AHEAD];
    fetch_c0(0);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) fetch(chunks[j], j);
    __syncthreads();
    for (int m0 = 0; m0 < n; m0 += AHEAD)
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
        const int m = m0 + j;
        const long long id = from + m * by;
        if (m >= n) break;
        const Chunk& c = chunks[j];
        Frag<CP> xs[DK / 32];
#pragma unroll
        for (int d = 0; d < NK; ++d) xs[d] = join(split<CP>(x[2 * d]), split<CP>(x[2 * d + 1]));
        f32x4 y[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) y[b] = BACK || unit_cols ? f32x4{0.f, 0.f, 0.f, 0.f} : c.y0[b];
#pragma unroll
        for (int d = 0; d < NK; ++d) {
            // (lane = step, values = channels of k)
            if constexpr (BACK) {
                Frag<RAW> a[4];
#pragma unroll
                for (int b = 0; b < 4; ++b) a[b] = L::tiles(lk, 16 * b, 32 * d, lane);
                mma_rows(a, xs[d], y);
            } else {
                Frag<CP> a[4];
#pragma unroll
                for (int b = 0; b < 4; ++b)
                    a[b] = join(read_turned<CP>(lw + (2 * d * 4 + b) * 256, PLANE, lane), read_turned<CP>(lw + ((2 * d + 1) * 4 + b) * 256, PLANE, lane));
                mma_rows(a, xs[d], y);
            }
        }
        if constexpr (!MAPS) {
            bf16_t* to = (BACK ? p.ds1 : p.s0) + id * z.state;
#pragma unroll
            for (int d = 0; d < NK; ++d) store_frag(to, cv * NK + d, planes<MADE>(xs[d]), lane);
        }
        if constexpr (!TWICE) __syncthreads();
        Half<CP> e[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) e[b] = split<CP>(y[b] * c.E[b]);
        const Frag<CP> e0 = join(e[0], e[1]), e1 = join(e[2], e[3]);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            x[d] = x[d] * c.end;
            if constexpr (BACK) x[d] += unit_cols ? f32x4{0.f, 0.f, 0.f, 0.f} : c0[d];
        }
        fetch_c0(m + 1);
#pragma unroll
        for (int d0 = 0; d0 < ND; d0 += ROWS) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                // (lane = channel of k, values = steps)
                Frag<BACK ? CP : RAW> a[ROWS];
                f32x4 t[ROWS];
#pragma unroll
                for (int i = 0; i < ROWS; ++i) {
                    const int d = d0 + i;
                    if constexpr (BACK) {
#pragma unroll
                        for (int q = 0; q < CP; ++q) {
                            const bf16x4 lo = *reinterpret_cast<const bf16x4*>(lw + q * PLANE + ((d * 4 + 2 * h) * 64 + lane) * 4);
                            const bf16x4 hi = *reinterpret_cast<const bf16x4*>(lw + q * PLANE + ((d * 4 + 2 * h + 1) * 64 + lane) * 4);
                            a[i].p[q] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                        }
                    } else {
                        a[i] = join(L::down(lk, 32 * h, 16 * d, lane), L::down(lk, 32 * h + 16, 16 * d, lane));
                    }
                    t[i] = x[d];
                }
                mma_rows(a, h ? e1 : e0, t);
#pragma unroll
                for (int i = 0; i < ROWS; ++i) x[d0 + i] = t[i];
            }
        }
        if constexpr (!MAPS && !BACK) {
            bf16_t* to = p.u + id * z.u;
            store_frag(to, cv * 2, join(split<MADE>(y[0]), split<MADE>(y[1])), lane);
            store_frag(to, cv * 2 + 1, join(split<MADE>(y[2]), split<MADE>(y[3])), lane);
        }
        fetch(chunks[j], m + AHEAD);
        if constexpr (TWICE) {
            const int other = m & 1 ? -delta_chain_values<T, DK, CP>() : delta_chain_values<T, DK, CP>();
            lw += other, lk += other;
        }
        __syncthreads();
    }
    if constexpr (MAPS) {
        const long long id = chain * (long long)(p.segments - 1) + segment;
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
    } else if (segment == p.segments - 1) {
        float* to = BACK ? p.gh0 : p.last;
        store_state<DK>(to ? to + state : nullptr, x, p.dk, p.dv, at, lane);
    }
}

// The state before every segment but the first, in the place of its predecessor's shift N: X = M X + N from segment to segment.  A workgroup has 16 columns
// of a chain, a wavefront 16 rows of them: its rows of the next segments' M are under way, X goes round through LDS (20 segments at 64 channels 16 us
// with one segment's under way, 13.5 with four).
template <typename T, int DK, bool BACK, int CP>
__global__ __launch_bounds__(DK * 4) void delta_join_k(DeltaArgs p) {
    // (maps of 128 x 128 are bound by their bytes: three segments ahead, the last one's map once or twice more, took 18 us for 16)
    constexpr int NK = DK / 32, AHEAD = DK == 128 ? 1 : 4;
    __shared__ __align__(16) bf16_t lx[2][NK * CP * 512];
    const int lane = threadIdx.x & 63, d = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), colv = p.dvp / 16;
    const unsigned id = (unsigned)p.first + blockIdx.x;
    const int chain = (int)(id / (unsigned)colv), cv = (int)(id - (unsigned)chain * colv);
    const DeltaSizes z(DK, p.dvp, 1, CP);
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
    // (behind the last segment's the last once more: loads on a condition would be waited for all together)
    struct Map {
        Frag<CP> m[NK];
        f32x4 n;
    };
    const int last = p.segments - 2;
    auto fetch = [&](Map& f, int s) {
        s = s < last ? s : last;
#pragma unroll
        for (int k = 0; k < NK; ++k) f.m[k] = load_frag<CP>(maps + s * z.map, d * NK + k, lane);
        f.n = load_at<f32x4>(shifts + s * z.shift, lane * 16);
    };
    Map ahead[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) fetch(ahead[j], j);
    for (int s0 = 0; s0 <= last; s0 += AHEAD)
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
        const int s = s0 + j;
        if (s > last) break;
        bf16_t* l = lx[s & 1];
        store_half(l, d / 2, d & 1, split<CP>(x), lane);
        __syncthreads();
        f32x4 t[NK];
#pragma unroll
        for (int k = 0; k < NK; ++k) t[k] = mma(ahead[j].m[k], load_frag<CP>(l, k, lane), k ? f32x4{0.f, 0.f, 0.f, 0.f} : ahead[j].n);
        x = t[0];
#pragma unroll
        for (int k = 1; k < NK; ++k) x += t[k];
        if (AHEAD > 1 || s < last) fetch(ahead[j], s + AHEAD);
        store_at(shifts + s * z.shift, lane * 16, x);
    }
}

}  // namespace pdw
