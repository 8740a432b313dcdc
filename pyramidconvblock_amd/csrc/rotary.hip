// Head norms with rotated positions: tokens of a workgroup, the launches of rotary.h's kernels, and the sum over workgroups for the weights'
// gradients.
#include "kernels.h"
#include "rotary.h"

namespace pdw {

int rotary_lanes_f32(int d, int P);
int rotary_lanes_f16(int d, int P);
int rotary_lanes_bf16(int d, int P);
void rotary_launch_f32(const RotaryArgs& p, unsigned grid, bool backward, hipStream_t s);
void rotary_launch_f16(const RotaryArgs& p, unsigned grid, bool backward, hipStream_t s);
void rotary_launch_bf16(const RotaryArgs& p, unsigned grid, bool backward, hipStream_t s);

// Workgroups that leave sums for the weights: four on every compute unit (with two, 50176 tokens of 8 and 4 heads of 64 channels in bf16 took 87 us instead of 73 then;
// with more their sums cost what they save).
constexpr long long kRotarySums = 1024;

// gw[s][c] = the sum over workgroups of parts[workgroup][s][c]: 16 columns a workgroup, 64 ranges of workgroups, in a fixed order.
template <typename T>
__global__ __launch_bounds__(1024) void rotary_sums_k(const float* __restrict__ parts, T* gq, T* gk, int workgroups, int d) {
    constexpr int CW = 16, Q = 64;
    __shared__ float red[Q][CW];
    const int cl = threadIdx.x % CW, q = threadIdx.x / CW, c = blockIdx.x * CW + cl;
    float a = 0.f;
    if (c < 2 * d)
        for (int g = q; g < workgroups; g += Q) a += parts[(long long)g * 2 * d + c];
    red[q][cl] = a;
    __syncthreads();
#pragma unroll
    for (int h = Q / 2; h > 0; h /= 2) {
        if (q < h) red[q][cl] += red[q + h][cl];
        __syncthreads();
    }
    if (q || c >= 2 * d) return;
    T* to = c < d ? gq : gk;
    if (to) to[c < d ? c : c - d] = from_f32<T>(red[0][cl]);
}

// Tokens of a workgroup: four rounds of rows (with two those gradients took 88 us, with eight 78), fewer where the call is small (512 workgroups at least;
// with 1024, of a few tokens each, one call of 1024 tokens took 8.9 us instead of 7.0), and angles that fit 16 KB.
static int rotary_tokens(const RotaryArgs& p, int lanes) {
    const int heads = p.heads[0] > p.heads[1] ? p.heads[0] : p.heads[1];
    long long t = (4 * (256 / lanes) + heads - 1) / heads;
    const long long even = p.N / 512, most = p.P ? 2048 / p.P : t;
    if (t > even) t = even;
    if (t > most) t = most;
    return t < 1 ? 1 : (int)t;
}

static int rotary_sums(const float* parts, void* gw, void* gkw, int workgroups, int d, int dtype, hipStream_t s) {
    const unsigned n = (2 * d + 15) / 16;
    if (dtype == kF32) rotary_sums_k<float><<<n, 1024, 0, s>>>(parts, (float*)gw, (float*)gkw, workgroups, d);
    else if (dtype == kF16) rotary_sums_k<f16_t><<<n, 1024, 0, s>>>(parts, (f16_t*)gw, (f16_t*)gkw, workgroups, d);
    else rotary_sums_k<bf16_t><<<n, 1024, 0, s>>>(parts, (bf16_t*)gw, (bf16_t*)gkw, workgroups, d);
    return check_launch("rotary_sums_k");
}

// The weights' gradients of a call without rows: sums of nothing.
int rotary_no_rows(void* gw, void* gkw, int d, int dtype, hipStream_t s) { return gw || gkw ? rotary_sums(nullptr, gw, gkw, 0, d, dtype, s) : 0; }

size_t rotary_workspace(int d) { return (size_t)kRotarySums * 2 * d * sizeof(float); }

int rotary_run(const RotaryArgs& in, bool backward, void* gw, void* gkw, void* workspace, size_t workspace_bytes, int dtype, hipStream_t s) {
    RotaryArgs p = in;
    const int lanes = dtype == kF32 ? rotary_lanes_f32(p.d, p.P) : dtype == kF16 ? rotary_lanes_f16(p.d, p.P) : rotary_lanes_bf16(p.d, p.P);
    p.TT = rotary_tokens(p, lanes);
    long long grid = (p.N + p.TT - 1) / p.TT;
    const bool sums = backward && (gw || gkw);
    if (sums && (!workspace || workspace_bytes < rotary_workspace(p.d)))
        return set_error("rotary: workspace too small (%zu of %zu bytes)", workspace_bytes, rotary_workspace(p.d)), 1;
    const long long most = sums ? kRotarySums : 4096;
    if (grid > most) grid = most;
    p.parts = sums ? (float*)workspace : nullptr;
    if (dtype == kF32) rotary_launch_f32(p, (unsigned)grid, backward, s);
    else if (dtype == kF16) rotary_launch_f16(p, (unsigned)grid, backward, s);
    else rotary_launch_bf16(p, (unsigned)grid, backward, s);
    if (int e = check_launch("rotary_k")) return e;
    return sums ? rotary_sums(p.parts, gw, gkw, (int)grid, p.d, dtype, s) : 0;
}

}  // namespace pdw
