// The gated linear recurrence: how time is cut into tiles and segments, the launches of scan.h's kernels, and the form for a
// single token.
#include "kernels.h"
#include "scan.h"

namespace pdw {

void scan_launch_f32(const ScanArgs& p, const ScanShape& shape, ScanPass pass, hipStream_t s);
void scan_launch_f16(const ScanArgs& p, const ScanShape& shape, ScanPass pass, hipStream_t s);
void scan_launch_bf16(const ScanArgs& p, const ScanShape& shape, ScanPass pass, hipStream_t s);

// Tiles of a chain, and segments of whole tiles, backward of pairs of tiles: where there are any, as many as 1024 workgroups of four wavefronts
// ask for, rounded up to whole tiles, so fewer workgroups ([2,50176,96]: 588 each way, two tiles and four).
struct ScanCut {
    ScanShape shape;
    long long strips, tiles, seg_tiles, segments;
};

static ScanCut scan_cut(long long rows, long long T, int I, ScanPass pass) {
    ScanCut c;
    c.shape = scan_shape(rows, T, I);
    c.strips = cdiv(I, c.shape.width());
    const int step = c.shape.tile(pass);
    c.tiles = (T + step - 1) / step;
    const long long columns = rows * c.strips;
    long long want = c.shape.segments ? (1024 + columns - 1) / columns : 1;
    if (want > c.tiles) want = c.tiles;
    if (want < 1) want = 1;
    c.seg_tiles = c.tiles ? (c.tiles + want - 1) / want : 1;
    const int whole = kMapSteps / c.shape.steps(pass);   // (a segment is whole batches of the kernel that composes its map)
    if (want > 1 && whole > 1) c.seg_tiles = (c.seg_tiles + whole - 1) / whole * whole;
    c.segments = c.tiles ? (c.tiles + c.seg_tiles - 1) / c.seg_tiles : 1;
    return c;
}

size_t scan_states_bytes(long long rows, long long T, int I) {
    return (size_t)(rows * scan_cut(rows, T, I, kScanBackward).tiles) * I * sizeof(float);
}

size_t scan_workspace(long long rows, long long T, int I, bool backward) {
    const ScanCut c = scan_cut(rows, T, I, backward ? kScanBackward : kScanForward);
    return c.segments > 1 ? (size_t)(c.segments * rows) * I * 2 * sizeof(float) : 0;
}

int scan_run(const ScanArgs& in, bool backward, void* workspace, size_t workspace_bytes, int dtype, hipStream_t s) {
    ScanArgs p = in;
    const ScanPass pass = backward ? kScanBackward : kScanForward;
    const ScanCut c = scan_cut(p.rows, p.T, p.I, pass);
    if (c.strips * p.rows * c.segments > 0x7fffffffLL || c.seg_tiles * c.shape.tile(pass) > 0x7fffffffLL)
        return set_error("scan: too many chains (%d x %d, %lld steps)", p.rows, p.I, p.T), 1;
    const size_t need = scan_workspace(p.rows, p.T, p.I, backward);
    if (need && (!workspace || workspace_bytes < need))
        return set_error("scan: workspace too small (%zu of %zu bytes)", workspace_bytes, need), 1;
    p.strips = (int)c.strips, p.tiles = (int)c.tiles, p.seg_tiles = (int)c.seg_tiles, p.segments = (int)c.segments;
    p.maps = (float*)workspace;
    long long far = 0;
    for (const ScanStrides& t : {p.xs, p.gs, p.gxs, p.ggs, p.dense}) {
        if (t.t < 0) far = 1LL << 40;
        if (t.t > far) far = t.t;
    }
    const long long step = c.shape.tile(pass), most = 0x3fffffffLL - p.I;   // elements: 32 bits of bytes
    p.near = far <= most / step, p.near_segments = far <= most / (step * c.seg_tiles);
    p.state_tiles = (int)scan_cut(p.rows, p.T, p.I, kScanBackward).tiles;
    if (dtype == kF32) scan_launch_f32(p, c.shape, pass, s);
    else if (dtype == kF16) scan_launch_f16(p, c.shape, pass, s);
    else scan_launch_bf16(p, c.shape, pass, s);
    return check_launch(backward ? "scan_bwd_k" : "scan_fwd_k");
}

// One step of every chain: y = new_state = a state + m x.  A thread has VEC neighbouring channels and no other thread touches them,
// so the new state may take the old one's place.  A few hundred kilobytes: launch latency is all there is to it.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void scan_step_k(const T* __restrict__ x, const T* __restrict__ g, const float* state, float* new_state,
                                                   T* __restrict__ y, long long n, int C, long long ldx, long long ldg, long long first) {
    const long long e = (first + blockIdx.x) * 256 + threadIdx.x;
    if (e >= n) return;
    const int per = C / VEC;
    const long long b = e / per;
    const int c = (int)(e - b * per) * VEC;
    const Piece<T, VEC> xr = load_any<T, VEC>(x + b * ldx + c), gr = load_any<T, VEC>(g + b * ldg + c);
    const Piece<float, VEC> h = load_any<float, VEC>(state + b * C + c);
    float a[VEC], m[VEC], out[VEC];
    gates<T, VEC>(gr, a, m);
#pragma unroll
    for (int v = 0; v < VEC; ++v) out[v] = __builtin_fmaf(a[v], h.v[v], m[v] * to_f32(xr.v[v]));
    store_any<float, VEC>(new_state + b * C + c, out);
    store_any<T, VEC>(y + b * C + c, out);
}

template <typename T>
static int step_launch(const void* x, const void* g, const float* state, float* new_state, void* y, long long B, int C,
                       long long ldx, long long ldg, hipStream_t s) {
    const bool wide = C % 4 == 0;
    const long long n = B * (C / (wide ? 4 : 1)), blocks = (n + 255) / 256;
    launch_parts(blocks, 256, [&](long long first, unsigned m) {
        if (wide) scan_step_k<T, 4><<<m, 256, 0, s>>>((const T*)x, (const T*)g, state, new_state, (T*)y, n, C, ldx, ldg, first);
        else scan_step_k<T, 1><<<m, 256, 0, s>>>((const T*)x, (const T*)g, state, new_state, (T*)y, n, C, ldx, ldg, first);
    });
    return check_launch("scan_step_k");
}

int scan_step_launch(const void* x, const void* g, const float* state, float* new_state, void* y, long long B, int C, long long ldx,
                     long long ldg, int dtype, hipStream_t s) {
    if (dtype == kF32) return step_launch<float>(x, g, state, new_state, y, B, C, ldx, ldg, s);
    if (dtype == kF16) return step_launch<f16_t>(x, g, state, new_state, y, B, C, ldx, ldg, s);
    return step_launch<bf16_t>(x, g, state, new_state, y, B, C, ldx, ldg, s);
}

}  // namespace pdw
