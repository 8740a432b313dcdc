// Norms over channels and gated residuals: how rows are cut into segments, the sum of their column sums, and the launches
// (kernels: row_norm.h, instantiated in row_norm_*.hip).
#include "kernels.h"
#include "row_norm.h"

namespace pdw {

int rows_lanes_f32(int C);
int rows_lanes_f16(int C);
int rows_lanes_bf16(int C);
void rows_launch_f32(const RowArgs& p, unsigned grid, bool backward, hipStream_t s);
void rows_launch_f16(const RowArgs& p, unsigned grid, bool backward, hipStream_t s);
void rows_launch_bf16(const RowArgs& p, unsigned grid, bool backward, hipStream_t s);

// Segments of an image's P rows, and rows of one, for `images` images: whole passes of a workgroup, and as many as give the chip the
// workgroups that measured best, a multiple of its 256 compute units: forward 2048, backward 512 (of eight wavefronts).  Rows of several
// wavefronts have a workgroup to themselves, and those of two to four wavefronts more of them (16-bit norm of 768 channels,
// forward: 2048 workgroups 4.4 TB/s, 4096 4.8; backward with the forward before it: 512 3.3, 1536 3.9; residual with its next norm, whose
// four column sums and what goes with them leave room for fewer: 512 3.1, 1024 3.9, 1536 3.5; of 1152 channels 512 3.6, 768 3.4).
static void plan_segments(long long images, long long P, int C, int dtype, bool backward, int sums, int* S, long long* L) {
    const int lanes = dtype == kF32 ? rows_lanes_f32(C) : rows_lanes_f16(C);
    long long G = 1, target = !backward ? 2048 : 512;
    if (lanes > 0) {
        G = (backward ? 512 : 256) / lanes;
    } else {
        const int pieces = cdiv(C, dtype == kF32 ? 4 : 8), waves = pieces > 512 ? 8 : cdiv(pieces, 64);
        if (!backward) target = waves <= 3 ? 4096 : 2048;
        else if (sums == 4) target = waves == 2 ? 1024 : 512;
        else target = waves == 2 ? 1536 : waves == 3 ? 1024 : waves == 4 ? 768 : 512;
    }
    long long want = (target + images - 1) / images;
    const long long passes = (P + G - 1) / G;
    if (want > passes) want = passes;
    if (want < 1) want = 1;
    *L = (passes + want - 1) / want * G;
    *S = (int)((P + *L - 1) / *L);
}

// The sums over segments, and what follows from them (row_norm.h).  One workgroup has 16 channels of one job: the residual's
// gradients of scale, weight and bias; the next norm's; or an image's gate row.  64 lanes a channel take every 64th segment,
// eight in flight: the pass is a few load latencies long.  The order of the additions is fixed.
struct ColsArgs {
    const float* parts;
    long long segments;
    const void *w, *b, *scale, *gate;
    void *gscale, *gw, *gb, *gw2, *gb2, *ggate;
    long long ldg;
    int C, S, sums, act, gate_rows;
    unsigned first;               // the launch's first workgroup (launch_parts)
    int branch_jobs, next_jobs;   // 1 or 0
};

template <typename T>
__global__ __launch_bounds__(1024) void rows_cols_k(ColsArgs p) {
    constexpr int CW = 16, Q = 64;
    __shared__ float2 red[Q][CW];
    const int blocks = (p.C + CW - 1) / CW;
    const unsigned block = p.first + blockIdx.x;
    const long long job = block / (unsigned)blocks;
    const int cl = threadIdx.x % CW, q = threadIdx.x / CW;
    const int c = (int)(block - job * blocks) * CW + cl;
    const bool image_job = job >= p.branch_jobs + p.next_jobs, next_job = !image_job && job >= p.branch_jobs;
    const long long image = job - p.branch_jobs - p.next_jobs;
    const long long s0 = image_job ? image * p.S : 0, s1 = image_job ? s0 + p.S : p.segments;
    const float* parts = p.parts + (next_job ? p.sums - 2 : 0) * (long long)p.C + c;
    const long long ld = (long long)p.sums * p.C;
    const bool weigh = !image_job && !next_job && p.gate_rows == 1;
    float a = 0.f, b = 0.f;
    if (c < p.C) {
        for (long long s = s0 + q; s < s1; s += 8 * Q) {
            float u[8], v[8], f[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const long long t = s + k * Q;
                u[k] = t < s1 ? parts[t * ld] : 0.f, v[k] = t < s1 ? parts[t * ld + p.C] : 0.f, f[k] = 1.f;
                if (weigh && t < s1) f[k] = to_f32(((const T*)p.gate)[(unsigned)t / (unsigned)p.S * p.ldg + c]);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float w = weigh && s + k * Q < s1 ? gate_act(f[k], p.act) : 1.f;
                a = __builtin_fmaf(w, u[k], a), b = __builtin_fmaf(w, v[k], b);
            }
        }
    }
    red[q][cl] = make_float2(a, b);
    __syncthreads();
#pragma unroll
    for (int h = Q / 2; h > 0; h /= 2) {
        if (q < h) red[q][cl] = make_float2(red[q][cl].x + red[q + h][cl].x, red[q][cl].y + red[q + h][cl].y);
        __syncthreads();
    }
    if (q != 0 || c >= p.C) return;
    a = red[0][cl].x, b = red[0][cl].y;
    if (next_job) {
        if (p.gw2) ((T*)p.gw2)[c] = from_f32<T>(a);
        if (p.gb2) ((T*)p.gb2)[c] = from_f32<T>(b);
        return;
    }
    const float w = p.w ? to_f32(((const T*)p.w)[c]) : 1.f, bias = p.b ? to_f32(((const T*)p.b)[c]) : 0.f;
    const float scale = p.scale ? to_f32(((const T*)p.scale)[c]) : 1.f;
    if (image_job) {
        float f, slope;
        gate_act_slope(to_f32(((const T*)p.gate)[image * p.ldg + c]), p.act, f, slope);
        ((T*)p.ggate)[image * p.C + c] = from_f32<T>(slope * scale * __builtin_fmaf(w, a, bias * b));
        return;
    }
    if (p.gscale) ((T*)p.gscale)[c] = from_f32<T>(__builtin_fmaf(w, a, bias * b));
    if (p.gw) ((T*)p.gw)[c] = from_f32<T>(scale * a);
    if (p.gb) ((T*)p.gb)[c] = from_f32<T>(scale * b);
}

static void launch_rows(const RowArgs& p, unsigned grid, bool backward, int dtype, hipStream_t s) {
    if (dtype == kF32) rows_launch_f32(p, grid, backward, s);
    else if (dtype == kF16) rows_launch_f16(p, grid, backward, s);
    else rows_launch_bf16(p, grid, backward, s);
}

static long long images_of(const RowArgs& p) { return p.gate_rows == 1 && p.N > 0 ? p.N / p.P : 1; }

// Where there is no gate row an image, all rows are one image.
static RowArgs cut(const RowArgs& in, bool backward, int dtype, long long* grid) {
    RowArgs p = in;
    const long long images = images_of(p);
    if (p.gate_rows != 1) p.P = p.N;
    plan_segments(images, p.P, p.C, dtype, backward, p.y && p.kind2 != kNormNone ? 4 : 2, &p.S, &p.L);
    *grid = images * p.S;
    return p;
}

int rows_forward_launch(const RowArgs& in, int dtype, hipStream_t s) {
    if (in.N == 0) return 0;
    long long grid;
    const RowArgs p = cut(in, false, dtype, &grid);
    if (grid > 0x7fffffffLL) return set_error("norm: too many images (%lld)", images_of(in)), 1;
    launch_rows(p, (unsigned)grid, false, dtype, s);
    return check_launch("rows_fwd_k");
}

size_t rows_backward_workspace(long long N, long long images, int C, int sums, int dtype) {
    if (N <= 0) return 0;
    int S;
    long long L;
    plan_segments(images, N / images, C, dtype, true, sums, &S, &L);
    return (size_t)images * S * sums * C * sizeof(float);
}

int rows_backward_launch(const RowArgs& in, void* gscale, void* gw, void* gb, void* gw2, void* gb2, void* workspace,
                         size_t workspace_bytes, int dtype, hipStream_t s) {
    const bool branch = in.y != nullptr, next = in.kind2 != kNormNone, image_gate = in.gate_rows == 1 && in.ggate && in.N > 0;
    const bool branch_sums = branch && (gscale || gw || gb), next_sums = next && (gw2 || gb2);
    const bool sums = branch_sums || next_sums || image_gate;
    const long long jobs = (long long)branch_sums + next_sums + (image_gate ? images_of(in) : 0), blocks = jobs * cdiv(in.C, 16);
    if (blocks > 0x7fffffffLL) return set_error("norm backward: too many images (%lld)", images_of(in)), 1;
    RowArgs p = in;
    long long grid = 0;
    p.parts = nullptr, p.S = 0;
    if (in.N > 0) {
        p = cut(in, true, dtype, &grid);
        if (grid > 0x7fffffffLL) return set_error("norm: too many images (%lld)", images_of(in)), 1;
        p.parts = sums ? (float*)workspace : nullptr;
        const size_t need = (size_t)grid * (branch && next ? 4 : 2) * p.C * sizeof(float);
        if (sums && (!workspace || workspace_bytes < need))
            return set_error("norm backward: workspace too small (%zu of %zu bytes)", workspace_bytes, need), 1;
        launch_rows(p, (unsigned)grid, true, dtype, s);
        if (int e = check_launch("rows_bwd_k")) return e;
    }
    if (!sums) return 0;
    ColsArgs c{};
    c.parts = (const float*)workspace, c.segments = grid;
    c.w = in.w, c.b = in.b, c.scale = in.scale, c.gate = in.gate, c.ldg = in.ldg;
    c.gscale = gscale, c.gw = gw, c.gb = gb, c.gw2 = gw2, c.gb2 = gb2, c.ggate = in.ggate;
    c.C = in.C, c.S = p.S, c.sums = branch && next ? 4 : 2, c.act = in.act, c.gate_rows = in.gate_rows;
    c.branch_jobs = branch_sums, c.next_jobs = next_sums;
    launch_parts(blocks, 1024, [&](long long first, unsigned n) {
        c.first = (unsigned)first;
        if (dtype == kF32) rows_cols_k<float><<<n, 1024, 0, s>>>(c);
        else if (dtype == kF16) rows_cols_k<f16_t><<<n, 1024, 0, s>>>(c);
        else rows_cols_k<bf16_t><<<n, 1024, 0, s>>>(c);
    });
    return check_launch("rows_cols_k");
}

}  // namespace pdw
