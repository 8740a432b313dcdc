// The gated linear recurrence  h_t = a_t h_(t-1) + m_t x_t,  a_t = sigmoid(g_t), m_t = 1 - a_t,  along the second axis of
// x[O][T][W][I], every one of the O x W x I chains by itself, and its gradients.
//
// A step maps h to a h + b; such maps compose associatively, (a, b) then (a', b') = (a a', a' b + b'), and a composition
// of a's in (0, 1) never grows, so a stretch of time can be cut anywhere: each piece is composed by itself, the pieces' maps are
// scanned, and each piece is run again from its own starting state.  Backwards, with d_t the gradient of h_t, the quantity handed from
// step t to step t - 1 is e_t = a_t d_t = a_t (gy_t + e_(t+1)): maps of the same kind with the same a, composed from the end.
//     gx_t = d_t m_t        gg_t = d_t (h_(t-1) - x_t) a_t m_t        (gradient of the initial state) = e_0
// The states h_(t-1) that gg needs are not kept: the forward leaves the 32-bit state before every tile, and the backward runs the tile
// from it again, in the same order, from x and g, which it reads anyway.
//
// A workgroup has a strip of channels (LC lanes of two channels) and walks over tiles of NW wavefronts x 64/LC lanes x K steps: a lane
// composes its K consecutive steps in registers, lanes and wavefronts exchange their maps (vector unit; LDS), and every lane runs its K
// steps from its state.  So x and g are read once.  Where there are too few strips to fill the chip, time is cut into segments of whole
// tiles: a first launch composes each segment's map (x and g are read once more for it), and the second starts each segment from the
// maps before it.
//
// All of it is in fp32.  No atomics: results are the same from call to call.
//
// What bounds it ([32,3136,128] bf16): instructions and their latencies, with eight wavefronts on a compute unit.  Forward a value takes 26
// (six of them the sigmoid, two of those at a quarter of the rate; an eighth of the tiles' steps lie behind a chain's end), 11 us of the
// 23 us kernel; backward 44, 18 us of 33; the rest is waiting, for loads and for the other wavefronts.  The tensors themselves would take 15 and 25 us from memory.  Forward and backward, replays of
// a captured pass of separate x and g (calls with x and g in halves of one tensor and other inputs each time: 65 us for the last of these): four
// channels a lane 107 us, two (half the exchanged values for as many steps) 87; stores of whole pieces and one branch a tile 78; strips
// of 16 channels without segments 73; lanes exchanged in the vector unit and one barrier for both scans of the backward 71; the next
// tile's loads under way 65; steps a lane that leave the last tile least empty 60.  From batches of 64 on it is memory: 3.8 ns for 1000
// values, 16 bytes each.
#pragma once
#include "common.h"
#include "gate_math.h"
#include "row_norm.h"

namespace pdw {

// Element (o, t, w, i) of a tensor is base[o * o + t * t + w * w + i].
struct ScanStrides {
    long long o, t, w;
};

struct ScanArgs {
    const void *x, *g, *gy;
    void *y, *gx, *gg;
    ScanStrides xs, gs, gxs, ggs, dense;   // dense: of y and gy
    const float *h0, *glast;            // [O][W][I], or null (0)
    float *last, *gh0;                  // [O][W][I], or null
    float* states;                      // [O * W][state_tiles][I]: the state before every tile of the backward, or null
    float* maps;                        // [segment][O * W][I] x (a, b): the segments' maps
    const int* lengths;                 // [O], or null (T)
    long long T;
    int rows, W, I;                     // rows = O * W
    int strips, tiles, segments, seg_tiles, state_tiles;
    unsigned blocks, first;             // workgroups in all, and the launch's first one (launch_parts)
    int reverse, near, near_segments;   // TilePtr's offsets fit, of a tile and of a segment
};

// Where a lane stands: its channels, and its steps within a tile.
template <int VEC, int LC, int NW, int K>
struct ScanLane {
    static constexpr int kSub = 64 / LC, kTile = NW * kSub * K;
    int lane, wave, c, sub;   // c: first channel
    bool on;
    __device__ __forceinline__ ScanLane(int strip, int I) {
        lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        c = (strip * LC + lane % LC) * VEC;
        on = c < I;
        if (c > I - VEC) c = I - VEC;   // the last lane overlaps the one before it: the same chains, the same values (I >= VEC)
        sub = wave * kSub + lane / LC;
    }
};

// The values of lanes l and l ^ D: that of the lower one and that of the upper one, in both.  Across 16 and 32 lanes an exchange in the
// vector unit, across eight a rotation of the row of 16, across four a permutation through LDS.
template <int D>
__device__ __forceinline__ void lane_pair(float x, int lane, float& lower, float& upper) {
    const unsigned u = __builtin_bit_cast(unsigned, x);
    unsigned lo, hi;
    if constexpr (D == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        lo = r[0], hi = r[1];
    } else if constexpr (D == 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        lo = r[0], hi = r[1];
    } else {
        const unsigned o = D == 8 ? (unsigned)__builtin_amdgcn_update_dpp(0, (int)u, 0x128, 0xf, 0xf, true) : (unsigned)__shfl_xor((int)u, D);
        lo = lane & D ? o : u, hi = lane & D ? u : o;
    }
    lower = __builtin_bit_cast(float, lo), upper = __builtin_bit_cast(float, hi);
}

// What a lane's map (a, b) becomes of a wavefront's: the composition of all (in every lane) and of those before the lane in the order of
// rising (BACK: falling) time.  Groups of LC lanes are pairs, pairs of pairs, and so on.
template <int VEC>
struct WaveMaps {
    float a[VEC], b[VEC];     // all
    float ea[VEC], eb[VEC];   // those before
};

template <int VEC, int LC, int D, bool BACK>
__device__ __forceinline__ void wave_level(WaveMaps<VEC>& w, const float (&la)[VEC], const float (&ha)[VEC], int lane) {
    const bool behind = BACK ? !(lane & D) : lane & D;   // the other half comes before this lane's
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        float lb, hb;
        lane_pair<D>(w.b[v], lane, lb, hb);
        const float fa = BACK ? ha[v] : la[v], fb = BACK ? hb : lb, sa = BACK ? la[v] : ha[v], sb = BACK ? lb : hb;
        w.b[v] = __builtin_fmaf(sa, fb, sb), w.a[v] = sa * fa;
        if (D == LC) {
            w.ea[v] = behind ? fa : 1.f, w.eb[v] = behind ? fb : 0.f;
        } else {
            const float eb = __builtin_fmaf(w.ea[v], fb, w.eb[v]), ea = w.ea[v] * fa;
            w.ea[v] = behind ? ea : w.ea[v], w.eb[v] = behind ? eb : w.eb[v];
        }
    }
}

// For one order of time (the other's b NULL), or for both, whose maps have the same a.
template <int VEC, int LC, int D, bool FORE, bool BACK>
__device__ __forceinline__ void wave_levels(WaveMaps<VEC>* fore, WaveMaps<VEC>* back, int lane) {
    if constexpr (D < 64) {
        float la[VEC], ha[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) lane_pair<D>(FORE ? fore->a[v] : back->a[v], lane, la[v], ha[v]);
        if constexpr (FORE) wave_level<VEC, LC, D, false>(*fore, la, ha, lane);
        if constexpr (BACK) wave_level<VEC, LC, D, true>(*back, la, ha, lane);
        wave_levels<VEC, LC, 2 * D, FORE, BACK>(fore, back, lane);
    }
}

// The wavefronts' maps: into LDS [NW][LC * VEC] (a, b), and, behind a barrier, through them: `carry`, the state at the tile's start (BACK: the
// gradient behind its end), is taken to its other side, and `start` is what this lane's steps start from.
template <int VEC, int LC>
__device__ __forceinline__ void wave_out(const WaveMaps<VEC>& w, float2* lds, int lane, int wave) {
    if (lane < LC) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) lds[(wave * LC + lane) * VEC + v] = make_float2(w.a[v], w.b[v]);
    }
}

template <int VEC, int LC, int NW, bool BACK>
__device__ __forceinline__ void wave_in(const WaveMaps<VEC>& m, float (&carry)[VEC], float (&start)[VEC], const float2* lds, int lane, int wave) {
    const int cl = lane % LC;
#pragma unroll 2   // (unrolled whole, the wavefronts' maps alone take 32 registers)
    for (int i = 0; i < NW; ++i) {
        const int w = BACK ? NW - 1 - i : i;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            if (w == wave) start[v] = carry[v];
            const float2 t = lds[(w * LC + cl) * VEC + v];
            carry[v] = __builtin_fmaf(t.x, carry[v], t.y);
        }
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) start[v] = __builtin_fmaf(m.ea[v], start[v], m.eb[v]);
}

// All of it for one order of time; lds: one buffer a call in turn.
template <int VEC, int LC, int NW, bool BACK>
__device__ __forceinline__ void scan_tile(WaveMaps<VEC>& m, float (&carry)[VEC], float (&start)[VEC], float2* lds, int lane, int wave) {
    wave_levels<VEC, LC, LC, !BACK, BACK>(&m, &m, lane);
    wave_out<VEC, LC>(m, lds, lane, wave);
    __syncthreads();
    wave_in<VEC, LC, NW, BACK>(m, carry, start, lds, lane, wave);
}

// The state that a segment starts from: `first` (the initial state, or the last one's gradient) through the maps of the segments
// before it (BACK: behind it).  The workgroup's lanes share them out as they share the steps of a tile.
template <int VEC, int LC, int NW, int K, bool BACK>
__device__ __forceinline__ void segment_start(const ScanArgs& p, int o, int seg, const ScanLane<VEC, LC, NW, K>& at,
                                              const float* first, float (&carry)[VEC], float2* lds) {
    constexpr int TS = NW * ScanLane<VEC, LC, NW, K>::kSub;
    const long long row = (long long)o * p.I + at.c, ld = (long long)p.rows * p.I;
#pragma unroll
    for (int v = 0; v < VEC; ++v) carry[v] = first && at.on ? first[row + v] : 0.f;
    const int n = BACK ? p.segments - 1 - seg : seg;   // maps to go through
    if (n == 0) return;
    const int each = (n + TS - 1) / TS;
    const int turn = BACK ? TS - 1 - at.sub : at.sub;   // this lane's place in the order of composition
    WaveMaps<VEC> m;
#pragma unroll
    for (int v = 0; v < VEC; ++v) m.a[v] = 1.f, m.b[v] = 0.f;
    for (int k = 0; k < each; ++k) {
        const int i = turn * each + k;
        if (i >= n || !at.on) break;
        const float2* t = reinterpret_cast<const float2*>(p.maps) + (BACK ? p.segments - 1 - i : i) * ld + row;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const float2 u = t[v];
            m.b[v] = __builtin_fmaf(u.x, m.b[v], u.y), m.a[v] *= u.x;
        }
    }
    float unused[VEC];
    scan_tile<VEC, LC, NW, BACK>(m, carry, unused, lds, at.lane, at.wave);
    __syncthreads();
}

// Position in memory of step s of a chain of `len` steps; steps behind its end stay where they are.
__device__ __forceinline__ long long scan_pos(long long s, long long len, int reverse) {
    return reverse && s < len ? len - 1 - s : s;
}

// What a workgroup's index says: its strip of channels, its row (o, w) and its segment; and its chains' length.  Neighbouring strips
// share cache lines, so those of a row go to one of the eight dies (workgroups go to them in turn), one after the other.
struct ScanWhere {
    int strip, row, o, w, seg;
    long long len;
    __device__ __forceinline__ ScanWhere(const ScanArgs& p) {
        const unsigned strips = p.strips, rows8 = p.blocks / strips & ~7u, block = p.first + blockIdx.x;
        unsigned rest;
        if (block < rows8 * strips) {
            const unsigned turn = block >> 3;
            strip = turn % strips, rest = turn / strips * 8 + (block & 7);
        } else {
            strip = block % strips, rest = block / strips;
        }
        row = rest % (unsigned)p.rows, seg = rest / (unsigned)p.rows;
        o = row / p.W, w = row - o * p.W;
        const long long n = p.lengths ? p.lengths[o] : p.T;
        len = n < 0 ? 0 : n > p.T ? p.T : n;
    }
    template <typename T>
    __device__ __forceinline__ T* base(T* t, const ScanStrides& s) const {
        return t + o * s.o + w * s.w;
    }
};

// Keeps the compiler from carrying what it has made of the pieces so far along with them.
template <typename T, int VEC, int K>
__device__ __forceinline__ void keep_packed(Piece<T, VEC> (&r)[K]) {
    if constexpr (sizeof(T) * VEC == 4) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            unsigned u = __builtin_bit_cast(unsigned, r[k]);
            asm("" : "+v"(u));
            r[k] = __builtin_bit_cast(Piece<T, VEC>, u);
        }
    }
}

// Steps of a lane that a segment's map is composed in at a time; segments are whole multiples of them.
constexpr int kMapSteps = 16;

// (a, m) of one piece of g
template <typename T, int VEC>
__device__ __forceinline__ void gates(const Piece<T, VEC>& g, float (&a)[VEC], float (&m)[VEC]) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) sigmoid_pair(to_f32(g.v[v]), a[v], m[v]);
}

// Where a lane's K steps of a tile of `tile` steps, from step `base` on, lie in one tensor: a base that all lanes share, a lane's
// offset in bytes (unsigned, 32 bits: the host has checked that a tile's extent fits), and the distance of a step.  A tile that is
// inside its chain is addressed this way, so that an address costs a lane nothing; others step by step, with 64 bits.
struct TilePtr {
    const char* shared;
    unsigned lane;
    long long step;
    // strip: the base of the chain's row, t: elements between positions, at: this lane's first step in the tile, c: its channel
    template <typename T>
    __device__ __forceinline__ TilePtr(const T* strip, long long t, long long base, int tile, long long len, int reverse, int at, int c) {
        const long long first = reverse ? len - base - tile : base;   // the tile's lowest position
        shared = (const char*)(strip + first * t);
        lane = ((unsigned)(reverse ? tile - 1 - at : at) * (unsigned)t + (unsigned)c) * (unsigned)sizeof(T);
        step = (reverse ? -t : t) * (long long)sizeof(T);
    }
    template <typename T>
    __device__ __forceinline__ T* of(int k) const {
        return (T*)(const_cast<char*>(shared) + k * step + lane);
    }
};

// A lane's K pieces of one tensor: all of them (whole), or those inside the chain, zeros for the others.
template <typename T, int VEC, int LC, int NW, int K>
__device__ __forceinline__ void load_steps(const T* strip, long long t, long long base, long long len, int reverse, bool whole,
                                           const ScanLane<VEC, LC, NW, K>& at, Piece<T, VEC> (&r)[K]) {
    if (whole) {
        const TilePtr p(strip, t, base, at.kTile, len, reverse, at.sub * K, at.c);
#pragma unroll
        for (int k = 0; k < K; ++k) r[k] = load_any<T, VEC>(p.of<const T>(k));
        return;
    }
    const long long s0 = base + (long long)at.sub * K;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if (s0 + k < len) r[k] = load_any<T, VEC>(strip + scan_pos(s0 + k, len, reverse) * t + at.c);
        else
#pragma unroll
            for (int v = 0; v < VEC; ++v) r[k].v[v] = from_f32<T>(0.f);
    }
}

// Stores a lane's K pieces; zeros at positions behind the chain's end.
template <typename T, int VEC, int LC, int NW, int K>
__device__ __forceinline__ void store_steps(T* strip, long long t, long long base, long long T_, long long len, int reverse, bool whole,
                                            const ScanLane<VEC, LC, NW, K>& at, const Piece<T, VEC> (&r)[K]) {
    if (!at.on) return;
    if (whole) {
        const TilePtr p(strip, t, base, at.kTile, len, reverse, at.sub * K, at.c);
#pragma unroll
        for (int k = 0; k < K; ++k) store_piece<T, VEC>(p.of<T>(k), r[k]);
        return;
    }
    const long long s0 = base + (long long)at.sub * K;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if (s0 + k >= T_) break;
        Piece<T, VEC> q = r[k];
        if (!(s0 + k < len)) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) q.v[v] = from_f32<T>(0.f);
        }
        store_piece<T, VEC>(strip + scan_pos(s0 + k, len, reverse) * t + at.c, q);
    }
}

// The map of every segment but the one that no other starts from (forward the last, BACK the first).  A lane composes a
// contiguous run of the segment's steps by itself, so the lanes exchange once, at the end.
template <typename T, int VEC, int LC, int NW, int TK, bool BACK>
__global__ __launch_bounds__(NW * 64) void scan_maps_k(ScanArgs p) {
    typedef ScanLane<VEC, LC, NW, TK> Lane;
    constexpr int K = kMapSteps;   // steps under way at once
    constexpr int TS = NW * Lane::kSub;
    __shared__ float2 lds[NW * LC * VEC];
    const ScanWhere my(p);
    const int seg = my.seg + (BACK ? 1 : 0);
    const Lane at(my.strip, p.I);
    const long long len = my.len;
    const T* other = my.base((const T*)(BACK ? p.gy : p.x), BACK ? p.dense : p.xs);
    const bool given = !BACK || p.gy;
    const long long ot = BACK ? p.dense.t : p.xs.t;
    const T* g = my.base((const T*)p.g, p.gs);
    const int steps = p.seg_tiles * Lane::kTile, run = steps / TS;   // the segment's steps and a lane's (a multiple of K)
    const long long first = (long long)seg * steps;
    WaveMaps<VEC> m;
#pragma unroll
    for (int v = 0; v < VEC; ++v) m.a[v] = 1.f, m.b[v] = 0.f;
    auto compose = [&](const Piece<T, VEC>& gp, const Piece<T, VEC>& op) {
        float a[VEC], q[VEC];
        gates<T, VEC>(gp, a, q);
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const float u = to_f32(op.v[v]);
            m.b[v] = BACK ? a[v] * (u + m.b[v]) : __builtin_fmaf(a[v], m.b[v], q[v] * u), m.a[v] *= a[v];
        }
    };
    if (p.near_segments && given && first + steps <= len) {
        const int end = at.sub * run + (BACK ? run - 1 : 0);   // the lane's first step in the order of composition
        const TilePtr pg(g, p.gs.t, first, steps, len, p.reverse, end, at.c), po(other, ot, first, steps, len, p.reverse, end, at.c);
        for (int i = 0; i < run; i += K) {
            Piece<T, VEC> xr[K], gr[K];
#pragma unroll
            for (int k = 0; k < K; ++k) gr[k] = load_any<T, VEC>(pg.of<const T>(BACK ? -i - k : i + k));
#pragma unroll
            for (int k = 0; k < K; ++k) xr[k] = load_any<T, VEC>(po.of<const T>(BACK ? -i - k : i + k));
#pragma unroll
            for (int k = 0; k < K; ++k) compose(gr[k], xr[k]);
        }
    } else {
        for (int i = 0; i < run; i += K) {
            Piece<T, VEC> xr[K], gr[K];
            const long long from = first + at.sub * run + (BACK ? run - 1 - i : i);
            if ((BACK ? from - K + 1 : from) >= len) continue;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const long long s = BACK ? from - k : from + k, t = scan_pos(s, len, p.reverse);
#pragma unroll
                for (int v = 0; v < VEC; ++v) xr[k].v[v] = gr[k].v[v] = from_f32<T>(0.f);
                if (s < len) gr[k] = load_any<T, VEC>(g + t * p.gs.t + at.c);
                if (s < len && given) xr[k] = load_any<T, VEC>(other + t * ot + at.c);
            }
#pragma unroll
            for (int k = 0; k < K; ++k)
                if ((BACK ? from - k : from + k) < len) compose(gr[k], xr[k]);
        }
    }
    float zero[VEC], one[VEC], unused[VEC];
    WaveMaps<VEC> product = m;
#pragma unroll
    for (int v = 0; v < VEC; ++v) zero[v] = 0.f, one[v] = 1.f, product.b[v] = 0.f;
    scan_tile<VEC, LC, NW, BACK>(m, zero, unused, lds, at.lane, at.wave);
    __syncthreads();
    scan_tile<VEC, LC, NW, BACK>(product, one, unused, lds, at.lane, at.wave);   // the maps' first halves, as what 1 becomes
    if (!at.on || at.sub != 0) return;
#pragma unroll
    for (int v = 0; v < VEC; ++v)
        reinterpret_cast<float2*>(p.maps)[((long long)seg * p.rows + my.row) * p.I + at.c + v] = make_float2(one[v], zero[v]);
}

// Workgroups of eight wavefronts, of which a compute unit has one, have the registers for the next tile's loads to be on their way while a
// tile is computed.
template <int NW>
constexpr bool scan_ahead() {
    return NW == 8;
}

template <typename T, int VEC, int LC, int NW, int K>
__global__ __launch_bounds__(NW * 64, scan_ahead<NW>() ? 2 : 4) void scan_fwd_k(ScanArgs p) {
    typedef ScanLane<VEC, LC, NW, K> Lane;
    constexpr int TS = NW * Lane::kSub;
    __shared__ float2 lds[2][NW * LC * VEC];
    const ScanWhere my(p);
    const int seg = my.seg;
    const Lane at(my.strip, p.I);
    const long long len = my.len;
    const T *x = my.base((const T*)p.x, p.xs), *g = my.base((const T*)p.g, p.gs);
    T* y = my.base((T*)p.y, p.dense);
    float carry[VEC];
    segment_start<VEC, LC, NW, K, false>(p, my.row, seg, at, p.h0, carry, lds[1]);
    const int t0 = seg * p.seg_tiles, t1 = t0 + p.seg_tiles < p.tiles ? t0 + p.seg_tiles : p.tiles;
    Piece<T, VEC> xr[K], gr[K];
    auto load = [&](int tile) {
        const long long base = (long long)tile * Lane::kTile;
        const bool whole = p.near && base + Lane::kTile <= len;
        load_steps(x, p.xs.t, base, len, p.reverse, whole, at, xr);
        load_steps(g, p.gs.t, base, len, p.reverse, whole, at, gr);
    };
    if (scan_ahead<NW>() && t0 < t1) load(t0);
    for (int tile = t0; tile < t1; ++tile) {
        const long long base = (long long)tile * Lane::kTile, s0 = base + (long long)at.sub * K;
        const bool whole = p.near && base + Lane::kTile <= len;
        if (!scan_ahead<NW>()) load(tile);
        float a[K][VEC], b[K][VEC], start[VEC];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            gates<T, VEC>(gr[k], a[k], b[k]);
#pragma unroll
            for (int v = 0; v < VEC; ++v) b[k][v] *= to_f32(xr[k].v[v]);
        }
        if (!whole) {
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (!(s0 + k < len))
#pragma unroll
                    for (int v = 0; v < VEC; ++v) a[k][v] = 1.f, b[k][v] = 0.f;
        }
        if (scan_ahead<NW>() && tile + 1 < t1) load(tile + 1);
        WaveMaps<VEC> m;
#pragma unroll
        for (int v = 0; v < VEC; ++v) m.a[v] = a[0][v], m.b[v] = b[0][v];
#pragma unroll
        for (int k = 1; k < K; ++k)
#pragma unroll
            for (int v = 0; v < VEC; ++v) m.b[v] = __builtin_fmaf(a[k][v], m.b[v], b[k][v]), m.a[v] *= a[k][v];
        scan_tile<VEC, LC, NW, false>(m, carry, start, lds[tile & 1], at.lane, at.wave);
        // (a tile is two of the backward's: the states before its first and its middle step)
        if (p.states && at.on && (at.sub == 0 || at.sub == TS / 2) && s0 < p.T) {
            float* st = p.states + ((long long)my.row * p.state_tiles + 2 * tile + (at.sub != 0)) * p.I + at.c;
#pragma unroll
            for (int v = 0; v < VEC; ++v) st[v] = start[v];
        }
        Piece<T, VEC> out[K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) start[v] = __builtin_fmaf(a[k][v], start[v], b[k][v]);
            out[k] = round_piece<T, VEC>(start);
        }
        store_steps(y, p.dense.t, base, p.T, len, p.reverse, whole, at, out);
    }
    if (p.last && seg == p.segments - 1 && at.on && at.sub == 0) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) p.last[(long long)my.row * p.I + at.c + v] = carry[v];
    }
}

template <typename T, int VEC, int LC, int NW, int K>
__global__ __launch_bounds__(NW * 64, scan_ahead<NW>() ? 2 : sizeof(T) == 2 && NW > 2 && LC > 8 ? 4 : 3) void scan_bwd_k(ScanArgs p) {
    typedef ScanLane<VEC, LC, NW, K> Lane;
    __shared__ float2 lds[2][2][NW * LC * VEC];
    const ScanWhere my(p);
    const int seg = my.seg;
    const Lane at(my.strip, p.I);
    const long long len = my.len;
    const T *x = my.base((const T*)p.x, p.xs), *g = my.base((const T*)p.g, p.gs), *gy = my.base((const T*)p.gy, p.dense);
    T *gx = my.base((T*)p.gx, p.gxs), *gg = my.base((T*)p.gg, p.ggs);
    float carry[VEC];
    segment_start<VEC, LC, NW, K, true>(p, my.row, seg, at, p.glast, carry, lds[1][0]);
    const int t0 = seg * p.seg_tiles, t1 = t0 + p.seg_tiles < p.tiles ? t0 + p.seg_tiles : p.tiles;
    Piece<T, VEC> xn[K], gn[K], gyn[K];
    float hn[VEC];
    auto load = [&](int tile) {
        const long long base = (long long)tile * Lane::kTile;
        const bool whole = p.near && base + Lane::kTile <= len;
        load_steps(g, p.gs.t, base, len, p.reverse, whole, at, gn);
        load_steps(gy, p.dense.t, base, p.gy ? len : 0, p.reverse, whole && p.gy, at, gyn);
        load_steps(x, p.xs.t, base, len, p.reverse, whole, at, xn);
#pragma unroll
        for (int v = 0; v < VEC; ++v) hn[v] = p.states[((long long)my.row * p.state_tiles + tile) * p.I + at.c + v];
    };
    if (scan_ahead<NW>() && t0 < t1) load(t1 - 1);
    for (int tile = t1 - 1; tile >= t0; --tile) {
        const long long base = (long long)tile * Lane::kTile, s0 = base + (long long)at.sub * K;
        const bool whole = p.near && base + Lane::kTile <= len;
        float a[K][VEC], m[K][VEC], e[VEC], hs[VEC], h[VEC];
        Piece<T, VEC> xr[K], gyr[K];
        if (!scan_ahead<NW>()) load(tile);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            gates<T, VEC>(gn[k], a[k], m[k]);
            xr[k] = xn[k], gyr[k] = gyn[k];
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) h[v] = hn[v];
        if (scan_ahead<NW>() && tile > t0) load(tile - 1);
        if (!whole) {
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (!(s0 + k < len))
#pragma unroll
                    for (int v = 0; v < VEC; ++v) a[k][v] = 1.f, m[k][v] = 0.f;
        }
        WaveMaps<VEC> back, fore;
#pragma unroll
        for (int v = 0; v < VEC; ++v) back.a[v] = 1.f, back.b[v] = fore.b[v] = 0.f;
#pragma unroll
        for (int k = K - 1; k >= 0; --k)
#pragma unroll
            for (int v = 0; v < VEC; ++v) back.b[v] = a[k][v] * (to_f32(gyr[k].v[v]) + back.b[v]), back.a[v] *= a[k][v];
#pragma unroll
        for (int v = 0; v < VEC; ++v) fore.a[v] = back.a[v];
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int v = 0; v < VEC; ++v) fore.b[v] = __builtin_fmaf(a[k][v], fore.b[v], m[k][v] * to_f32(xr[k].v[v]));
        // (kept as they were loaded, and converted again where they are used: 16 registers instead of 32)
        keep_packed(xr), keep_packed(gyr);
        wave_levels<VEC, LC, LC, true, true>(&fore, &back, at.lane);
        wave_out<VEC, LC>(fore, lds[tile & 1][0], at.lane, at.wave), wave_out<VEC, LC>(back, lds[tile & 1][1], at.lane, at.wave);
        __syncthreads();
        wave_in<VEC, LC, NW, false>(fore, h, hs, lds[tile & 1][0], at.lane, at.wave);
        wave_in<VEC, LC, NW, true>(back, carry, e, lds[tile & 1][1], at.lane, at.wave);
        float hx[K][VEC];   // h_(t-1) - x_t
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                hx[k][v] = hs[v] - to_f32(xr[k].v[v]);
                hs[v] = __builtin_fmaf(a[k][v], hs[v], m[k][v] * to_f32(xr[k].v[v]));
            }
        Piece<T, VEC> ox[K], og[K];
#pragma unroll
        for (int k = K - 1; k >= 0; --k) {
            float fx[VEC], fg[VEC];
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const float d = to_f32(gyr[k].v[v]) + e[v];
                fx[v] = d * m[k][v];
                e[v] = a[k][v] * d;
                fg[v] = fx[v] * a[k][v] * hx[k][v];
            }
            ox[k] = round_piece<T, VEC>(fx), og[k] = round_piece<T, VEC>(fg);
        }
        if (p.gx) store_steps(gx, p.gxs.t, base, p.T, len, p.reverse, whole, at, ox);
        if (p.gg) store_steps(gg, p.ggs.t, base, p.T, len, p.reverse, whole, at, og);
    }
    if (p.gh0 && seg == 0 && at.on && at.sub == 0) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) p.gh0[(long long)my.row * p.I + at.c + v] = carry[v];
    }
}

enum ScanPass { kScanForward, kScanBackward };

// How a call is cut: channels of a lane, lanes of a strip, wavefronts of a workgroup, whether time is cut into segments, and a lane's steps
// of a tile backward, up to eight (three tensors and two scans are held); forward it has twice as many.
struct ScanShape {
    int vec, lanes, waves;
    bool segments;
    int back;
    int width() const { return vec * lanes; }
    int steps(ScanPass pass) const { return pass == kScanForward ? 2 * back : back; }
    int tile(ScanPass pass) const { return waves * (64 / lanes) * steps(pass); }
};

// Without segments x and g are read once, in one launch, as long as there are workgroups for the chip: of eight wavefronts one on each of
// the 256 compute units, of four wavefronts four on each.  Strips are of 32 channels, of 16 where only those come near 256.
// Microseconds, forward and backward, replays of a captured pass with eight steps a lane throughout, [B,3136,128] bf16 (strips of 32: 4 B, of 16: 8 B):
//     B     32 channels, 8 wavefronts     4 wavefronts     16 channels, 8 wavefronts     segments
//     32                81                    118                     65                    78
//     38                82                    121                    107                    90
//     64               101                    145                    130                   133
//     96               182                    195                    207                   208
//     128              207                    219                    282                   276
// and [275,784,128]: 155, 126, 186, 154.  As many wavefronts as a chain's steps need, at most; a chain of up to 32 steps has a strip
// of 64 channels.  A chain without segments ends with a tile that costs as much as a whole one: of eight, seven and six steps a lane the
// number is taken that has the fewest steps in all, with three for a tile's exchange.  A pass of both directions with eight alone and with
// this rule: [32,3136,128] 65, 60 us (tiles of 896 steps forward instead of 1024), [64,3136,128] 99, 95, [275,784,128] 127, 120,
// [275,196,128] 46, 43, [64,1800,128] 61, 61 (six steps there would take 62).
inline ScanShape scan_shape(long long rows, long long T, int I) {
    if (I < 2) return {1, 4, 4, true, 8};
    const long long wide = rows * cdiv(I, 32), narrow = rows * cdiv(I, 16);
    const bool segments = narrow < 208;
    const int lanes = T <= 32 ? 32 : !segments && narrow <= 256 ? 8 : 16;
    const int most = segments || (wide > 256 && wide < 352) || wide > 512 ? 4 : 8;
    int waves = 1;
    while (waves < most && waves * (64 / lanes) * 16 < T) waves *= 2;
    ScanShape shape{2, lanes, waves, segments, 8};
    auto cost = [&](int back) {
        const long long tile = (long long)waves * (64 / lanes) * back;
        return (T + tile - 1) / tile * (back + 3) + (T + 2 * tile - 1) / (2 * tile) * (2 * back + 3);
    };
    if (!segments)
        for (int back : {7, 6})
            if (cost(back) < cost(shape.back)) shape.back = back;
    return shape;
}

template <typename T, int VEC, int LC, int NW, int BACK>
void scan_launch(const ScanArgs& p, ScanPass pass, hipStream_t s) {
    const unsigned columns = (unsigned)p.strips * (unsigned)p.rows;
    ScanArgs q = p;
    if constexpr (BACK == 8 && NW <= 4 && (LC == 16 || VEC == 1)) {   // (the shapes that are cut into segments)
        if (p.segments > 1) {
            q.blocks = columns * (unsigned)(p.segments - 1);
            launch_parts(q.blocks, NW * 64, [&](long long first, unsigned n) {
                q.first = (unsigned)first;
                if (pass == kScanForward) scan_maps_k<T, VEC, LC, NW, 2 * BACK, false><<<n, NW * 64, 0, s>>>(q);
                else scan_maps_k<T, VEC, LC, NW, BACK, true><<<n, NW * 64, 0, s>>>(q);
            });
        }
    }
    q.blocks = columns * (unsigned)p.segments;
    launch_parts(q.blocks, NW * 64, [&](long long first, unsigned n) {
        q.first = (unsigned)first;
        if (pass == kScanForward) scan_fwd_k<T, VEC, LC, NW, 2 * BACK><<<n, NW * 64, 0, s>>>(q);
        else scan_bwd_k<T, VEC, LC, NW, BACK><<<n, NW * 64, 0, s>>>(q);
    });
}

template <typename T, int LC, int BACK>
void scan_waves(const ScanArgs& p, const ScanShape& shape, ScanPass pass, hipStream_t s) {
    if (shape.waves == 1) scan_launch<T, 2, LC, 1, BACK>(p, pass, s);
    else if (shape.waves == 2) scan_launch<T, 2, LC, 2, BACK>(p, pass, s);
    else if (shape.waves == 4) scan_launch<T, 2, LC, 4, BACK>(p, pass, s);
    else scan_launch<T, 2, LC, 8, BACK>(p, pass, s);
}

template <typename T, int BACK>
void scan_lanes(const ScanArgs& p, const ScanShape& shape, ScanPass pass, hipStream_t s) {
    if (shape.lanes == 32) scan_launch<T, 2, 32, 1, BACK>(p, pass, s);   // (one wavefront holds 32 steps)
    else if (shape.lanes == 16) scan_waves<T, 16, BACK>(p, shape, pass, s);
    else scan_waves<T, 8, BACK>(p, shape, pass, s);
}

template <typename T>
void scan_dispatch(const ScanArgs& p, const ScanShape& shape, ScanPass pass, hipStream_t s) {
    if (shape.vec == 1) scan_launch<T, 1, 4, 4, 8>(p, pass, s);
    else if (shape.back == 8) scan_lanes<T, 8>(p, shape, pass, s);
    else if (shape.back == 7) scan_lanes<T, 7>(p, shape, pass, s);
    else scan_lanes<T, 6>(p, shape, pass, s);
}

}  // namespace pdw
