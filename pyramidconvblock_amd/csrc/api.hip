// C ABI of libpdw.so (declared in include/pdw.h): argument validation and dispatch to
// the kernel launchers.  No allocation, no synchronisation; the only state is the per-thread
// error text here, the per-thread list of deferred summations (dwconv_direct.hip), the
// once-per-process LDS-limit set-up next to each large kernel's launcher, the bounded per-shape
// launch-plan caches (dwconv_fwd2.h, dwconv_bwd3.h, and PlanCache of tile_common.h in dwconv_tz.h, dwconv_tiled.h,
// dwconv_wgrad_tiled.h: a std::map behind a mutex each, emptied at kPlanCacheMax entries) and the per-device address of the static scratch array.
#include <stdarg.h>
#include <stdio.h>

#include <mutex>

#include "../../include/pdw.h"
#include "common.h"
#include "kernels.h"
#include "pool_branch.h"
#include "reduce_parts.h"
#include "delta_common.h"
#include "rotary.h"
#include "scan.h"

namespace pdw {

static thread_local char g_err[512] = "";

void set_error(const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof(g_err), fmt, ap);
    va_end(ap);
}

int check_launch(const char* what) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        set_error("%s: launch failed: %s", what, hipGetErrorString(e));
        return 2;
    }
    return 0;
}

static bool valid_dtype(int dtype) { return dtype == kF32 || dtype == kF16 || dtype == kBF16; }

static int check_conv(const char* fn, const void* a, const void* b, const void* c, int B, int H, int W, int C, int KH,
                      int KW, int SH, int SW, int PH, int PW, int DH, int DW, int dtype) {
    if (!valid_dtype(dtype)) return set_error("%s: unknown dtype %d", fn, dtype), 1;
    if (B < 0 || H < 1 || W < 1 || C < 1 || KH < 1 || KW < 1)
        return set_error("%s: bad extents B=%d H=%d W=%d C=%d KH=%d KW=%d", fn, B, H, W, C, KH, KW), 1;
    if (SH < 1 || SW < 1 || DH < 1 || DW < 1 || PH < 0 || PW < 0)
        return set_error("%s: bad stride/padding/dilation (%d,%d)/(%d,%d)/(%d,%d)", fn, SH, SW, PH, PW, DH, DW), 1;
    if (B > 0 && (!a || !b || !c)) return set_error("%s: null pointer", fn), 1;
    return 0;
}

static int check_rows(const char* fn, long long N, int C, int kind, int next_kind, int act, int dtype) {
    if (!valid_dtype(dtype)) return set_error("%s: unknown dtype %d", fn, dtype), 1;
    if (N < 0 || C < 1 || C > PDW_NORM_MAX_CHANNELS)
        return set_error("%s: need N >= 0 and 1 <= C <= %d (N=%lld C=%d)", fn, PDW_NORM_MAX_CHANNELS, N, C), 1;
    for (int k : {kind, next_kind})
        if (k < kNormNone || k > kNormLayer) return set_error("%s: unknown norm %d", fn, k), 1;
    if (act < kActNone || act > kActSilu) return set_error("%s: unknown activation %d", fn, act), 1;
    return 0;
}

// The gate of a residual: a row for P rows, or a value for each.
static int check_gate(const char* fn, const void* gate, long long N, int C, long long P, long long* ldgate) {
    if (!gate) return 0;
    if (P < 1 || N % P) return set_error("%s: %lld rows are no multiple of P=%lld", fn, N, P), 1;
    if (*ldgate == 0) *ldgate = C;
    if (*ldgate < 0) return set_error("%s: ldgate=%lld", fn, *ldgate), 1;
    return 0;
}

static int check_scan(const char* fn, const void* x, const void* g, const long long* xs, const long long* gs, int O, long long T,
                      int W, int I, int dtype) {
    if (!valid_dtype(dtype)) return set_error("%s: unknown dtype %d", fn, dtype), 1;
    if (O < 0 || T < 0 || W < 0 || I < 0 || (long long)O * W > 0x7fffffffLL || T > 0x7fffffffLL)
        return set_error("%s: bad extents O=%d T=%lld W=%d I=%d", fn, O, T, W, I), 1;
    if (O > 0 && T > 0 && W > 0 && I > 0 && (!x || !g || !xs || !gs)) return set_error("%s: null pointer", fn), 1;
    return 0;
}

static int check_resample(const char* fn, const void* a, const void* b, int B, int H, int W, int C, int h, int w,
                          int dtype) {
    if (!valid_dtype(dtype)) return set_error("%s: unknown dtype %d", fn, dtype), 1;
    if (B < 0 || H < 1 || W < 1 || C < 1 || h < 1 || w < 1)
        return set_error("%s: bad extents B=%d H=%d W=%d C=%d h=%d w=%d", fn, B, H, W, C, h, w), 1;
    if (B > 0 && (!a || !b)) return set_error("%s: null pointer", fn), 1;
    if ((long long)H * h >= 0x7fffffffLL || (long long)W * w >= 0x7fffffffLL)
        return set_error("%s: extents too large", fn), 1;
    return 0;
}

// Scratch of the entry point that allocates nothing (pdw_dwconv_wgrad_static): one copy of this array lives on every
// device the library is loaded on, at that device's own address.  The name is a host-side stand-in; device
// code and HIP calls get the address hipGetSymbolAddress returns for the current device.
constexpr size_t kStaticScratchBytes = (size_t)32 << 20;
static __device__ __align__(256) unsigned char scratch[kStaticScratchBytes];

constexpr int kMaxDevices = 64;
static std::mutex g_scratch_mu;
static void* g_scratch_ptr[kMaxDevices] = {};

// Address of `scratch` on the current device, looked up once per device (with that device current).
static int static_scratch(const char* fn, void** out) {
    int dev = -1;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return set_error("%s: hipGetDevice: %s", fn, hipGetErrorString(e)), 2;
    if (dev < 0 || dev >= kMaxDevices) return set_error("%s: device index %d not supported", fn, dev), 2;
    std::lock_guard<std::mutex> lock(g_scratch_mu);
    if (!g_scratch_ptr[dev]) {
        void* p = nullptr;
        e = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch));
        if (e != hipSuccess || !p)
            return set_error("%s: hipGetSymbolAddress(scratch): %s", fn, hipGetErrorString(e)), 2;
        g_scratch_ptr[dev] = p;
    }
    *out = g_scratch_ptr[dev];
    return 0;
}

}  // namespace pdw

using namespace pdw;

extern "C" {

int pdw_version(void) { return 7; }

const char* pdw_last_error(void) { return g_err; }

int pdw_conv_out_size(int in, int k, int stride, int pad, int dil) {
    if (in < 1 || k < 1 || stride < 1 || dil < 1 || pad < 0) return 0;
    return conv_out_size(in, k, stride, pad, dil);
}

int pdw_dwconv_fwd(const void* x, const void* w, void* y, int B, int H, int W, int C, int KH, int KW, int SH, int SW,
                   int PH, int PW, int DH, int DW, int dtype, void* stream) {
    if (int e = check_conv("pdw_dwconv_fwd", x, w, y, B, H, W, C, KH, KW, SH, SW, PH, PW, DH, DW, dtype)) return e;
    if (B == 0 || conv_out_size(H, KH, SH, PH, DH) == 0 || conv_out_size(W, KW, SW, PW, DW) == 0) return 0;
    if (SH == 1 && SW == 1 && DH == 1 && DW == 1) {
        const int r = dwconv_tiled_launch(x, w, y, B, H, W, C, KH, KW, PH, PW, false, dtype, (hipStream_t)stream);
        if (r != -1) return r;
    }
    return dwconv_fwd_direct_launch(x, w, y, B, H, W, C, KH, KW, SH, SW, PH, PW, DH, DW, dtype, (hipStream_t)stream);
}

int pdw_dwconv_fwd_pool(const void* x, const void* w, void* y, void* xp, int B, int H, int W, int C, int KH, int KW,
                        int SH, int SW, int PH, int PW, int DH, int DW, int h, int wp, int dtype, void* stream) {
    if (int e = check_conv("pdw_dwconv_fwd_pool", x, w, y, B, H, W, C, KH, KW, SH, SW, PH, PW, DH, DW, dtype)) return e;
    if (int e = check_resample("pdw_dwconv_fwd_pool", x, xp, B, H, W, C, h, wp, dtype)) return e;
    if (B == 0) return 0;
    const int OH = conv_out_size(H, KH, SH, PH, DH), OW = conv_out_size(W, KW, SW, PW, DW);
    if (OH > 0 && OW > 0 && SH == 1 && SW == 1 && DH == 1 && DW == 1 && H == 2 * h && W == 2 * wp) {
        const int r = dwconv_tiled_launch(x, w, y, B, H, W, C, KH, KW, PH, PW, false, dtype, (hipStream_t)stream, nullptr,
                                          xp);
        if (r != -1) return r;
    }
    if (int e = pdw_dwconv_fwd(x, w, y, B, H, W, C, KH, KW, SH, SW, PH, PW, DH, DW, dtype, stream)) return e;
    return avgpool_fwd_launch(x, xp, B, H, W, C, h, wp, dtype, (hipStream_t)stream);
}

int pdw_dwconv_fwd_gate(const void* x, const void* w, void* y, void* xp, int B, int H, int W, int C, int K, int pad,
                        int ldy, int ych, int dtype, void* stream) {
    if (!valid_dtype(dtype)) return set_error("pdw_dwconv_fwd_gate: unknown dtype %d", dtype), 1;
    if (B < 0 || H < 1 || W < 1 || C < 2 || K < 1 || pad < 0)
        return set_error("pdw_dwconv_fwd_gate: bad extents B=%d H=%d W=%d C=%d K=%d pad=%d", B, H, W, C, K, pad), 1;
    if (ldy == 0) ldy = C / 2;
    if ((C & 1) || ych < 0 || ldy < ych + C / 2)
        return set_error("pdw_dwconv_fwd_gate: need even C and ych + C/2 <= ldy (C=%d ldy=%d ych=%d)", C, ldy, ych), 1;
    if (B > 0 && (!x || !w || !y)) return set_error("pdw_dwconv_fwd_gate: null pointer"), 1;
    if (B == 0) return 0;
    const int r = dwconv_gate_launch(x, w, y, xp, B, H, W, C, K, pad, pad, ldy, ych, dtype, (hipStream_t)stream);
    if (r == -1)
        return set_error("pdw_dwconv_fwd_gate: B=%d H=%d W=%d C=%d K=%d pad=%d dtype=%d not covered by the fused kernel", B,
                         H, W, C, K, pad, dtype), 3;
    return r;
}

int pdw_dwconv_dgrad(const void* gy, const void* w, void* dx, int B, int H, int W, int C, int KH, int KW, int SH,
                     int SW, int PH, int PW, int DH, int DW, int dtype, void* stream) {
    if (int e = check_conv("pdw_dwconv_dgrad", gy, w, dx, B, H, W, C, KH, KW, SH, SW, PH, PW, DH, DW, dtype)) return e;
    if (B == 0) return 0;
    if (SH == 1 && SW == 1 && DH == 1 && DW == 1 && PH <= KH - 1 && PW <= KW - 1) {
        // dx = correlation of gy with the 180-degree rotated filter at padding k-1-p
        const int OH = conv_out_size(H, KH, 1, PH, 1), OW = conv_out_size(W, KW, 1, PW, 1);
        if (OH > 0 && OW > 0) {
            const int r = dwconv_tiled_launch(gy, w, dx, B, OH, OW, C, KH, KW, KH - 1 - PH, KW - 1 - PW, true, dtype,
                                              (hipStream_t)stream);
            if (r != -1) return r;
        }
    }
    return dwconv_dgrad_direct_launch(gy, w, dx, B, H, W, C, KH, KW, SH, SW, PH, PW, DH, DW, dtype,
                                      (hipStream_t)stream);
}

int pdw_dwconv_dgrad_addpool(const void* gy, const void* w, const void* gp, void* dx, int B, int H, int W, int C, int KH,
                             int KW, int SH, int SW, int PH, int PW, int DH, int DW, int h, int wp, int dtype,
                             void* stream) {
    if (int e = check_conv("pdw_dwconv_dgrad_addpool", gy, w, dx, B, H, W, C, KH, KW, SH, SW, PH, PW, DH, DW, dtype))
        return e;
    if (int e = check_resample("pdw_dwconv_dgrad_addpool", gp, dx, B, H, W, C, h, wp, dtype)) return e;
    if (B == 0) return 0;
    if (SH == 1 && SW == 1 && DH == 1 && DW == 1 && PH <= KH - 1 && PW <= KW - 1) {
        const int OH = conv_out_size(H, KH, 1, PH, 1), OW = conv_out_size(W, KW, 1, PW, 1);
        if (OH > 0 && OW > 0 && dtype == kF32 && KH == KW) {   // any ratio
            const int r = dwconv_f32t_launch(gy, w, gp, dx, B, OH, OW, C, KW, KH - 1 - PH, KW - 1 - PW, true, h, wp,
                                             (hipStream_t)stream);
            if (r != -1) return r;
        } else if (OH > 0 && OW > 0 && H == 2 * h && W == 2 * wp) {
            const int r = dwconv_tiled_launch(gy, w, dx, B, OH, OW, C, KH, KW, KH - 1 - PH, KW - 1 - PW, true, dtype,
                                              (hipStream_t)stream, gp);
            if (r != -1) return r;
        }
    }
    if (int e = pdw_dwconv_dgrad(gy, w, dx, B, H, W, C, KH, KW, SH, SW, PH, PW, DH, DW, dtype, stream)) return e;
    return avgpool_bwd_launch(gp, dx, B, H, W, C, h, wp, 1, dtype, (hipStream_t)stream);
}

int pdw_sum_parts(const float* parts, void* out, int nparts, long long n, int dtype, void* stream) {
    if (!valid_dtype(dtype)) return set_error("pdw_sum_parts: unknown dtype %d", dtype), 1;
    if (nparts < 1 || n < 0 || n > 0x7fffffffLL) return set_error("pdw_sum_parts: bad extents nparts=%d n=%lld", nparts, n), 1;
    if (n == 0) return 0;
    if (!parts || !out) return set_error("pdw_sum_parts: null pointer"), 1;
    switch (dtype) {
        case kF32: return wgrad_reduce_launch<float>(parts, out, nparts, (int)n, (hipStream_t)stream);
        case kF16: return wgrad_reduce_launch<f16_t>(parts, out, nparts, (int)n, (hipStream_t)stream);
        default: return wgrad_reduce_launch<bf16_t>(parts, out, nparts, (int)n, (hipStream_t)stream);
    }
}

int pdw_reduce_defer_begin(void) { return reduce_defer_begin(); }

int pdw_reduce_defer_flush(void* stream) { return reduce_defer_flush((hipStream_t)stream); }

size_t pdw_dwconv_wgrad_workspace_bytes(int B, int H, int W, int C, int KH, int KW, int SH, int SW, int PH, int PW,
                                        int DH, int DW, int dtype) {
    if (check_conv("pdw_dwconv_wgrad_workspace_bytes", "", "", "", B, H, W, C, KH, KW, SH, SW, PH, PW, DH, DW, dtype))
        return 0;
    size_t need = dwconv_wgrad_direct_workspace(B, H, W, C, KH, KW, SH, SW, PH, PW, DH, DW);
    if (SH == 1 && SW == 1 && DH == 1 && DW == 1) {
        const size_t t = dwconv_wgrad_tiled_workspace(B, H, W, C, KH, KW, PH, PW, dtype);
        if (t > need) need = t;
    }
    return need;
}

int pdw_dwconv_wgrad(const void* x, const void* gy, void* dw, void* workspace, size_t workspace_bytes, int B, int H,
                     int W, int C, int KH, int KW, int SH, int SW, int PH, int PW, int DH, int DW, int dtype,
                     void* stream) {
    if (int e = check_conv("pdw_dwconv_wgrad", x, gy, dw, B, H, W, C, KH, KW, SH, SW, PH, PW, DH, DW, dtype)) return e;
    if (!dw) return set_error("pdw_dwconv_wgrad: null dw"), 1;
    const size_t need = pdw_dwconv_wgrad_workspace_bytes(B, H, W, C, KH, KW, SH, SW, PH, PW, DH, DW, dtype);
    if (!workspace || workspace_bytes < need)
        return set_error("pdw_dwconv_wgrad: workspace of %zu bytes given, %zu needed", workspace_bytes, need), 1;
    if (B > 0 && SH == 1 && SW == 1 && DH == 1 && DW == 1) {
        const int r = dwconv_wgrad_tiled_launch(x, gy, dw, workspace, B, H, W, C, KH, KW, PH, PW, dtype,
                                                (hipStream_t)stream);
        if (r != -1) return r;
    }
    return dwconv_wgrad_direct_launch(x, gy, dw, workspace, B, H, W, C, KH, KW, SH, SW, PH, PW, DH, DW, dtype,
                                      (hipStream_t)stream);
}

int pdw_dwconv_bwd(const void* gy, const void* w, const void* x, void* dx, void* dw, void* workspace, size_t workspace_bytes, int B, int H,
                   int W, int C, int KH, int KW, int SH, int SW, int PH, int PW, int DH, int DW, int dtype, void* stream) {
    if (int e = check_conv("pdw_dwconv_bwd", gy, w, dx, B, H, W, C, KH, KW, SH, SW, PH, PW, DH, DW, dtype)) return e;
    if (int e = check_conv("pdw_dwconv_bwd", x, gy, dw, B, H, W, C, KH, KW, SH, SW, PH, PW, DH, DW, dtype)) return e;
    if (!dw) return set_error("pdw_dwconv_bwd: null dw"), 1;
    const size_t need = pdw_dwconv_wgrad_workspace_bytes(B, H, W, C, KH, KW, SH, SW, PH, PW, DH, DW, dtype);
    if (!workspace || workspace_bytes < need)
        return set_error("pdw_dwconv_bwd: workspace of %zu bytes given, %zu needed", workspace_bytes, need), 1;
    if (B > 0 && SH == 1 && SW == 1 && DH == 1 && DW == 1 && KH == KW && (KH & 1) && PH == KH / 2 && PW == PH) {
        const int r = dwconv_bwd3_launch(gy, w, nullptr, dx, x, dw, workspace, nullptr, nullptr, nullptr, nullptr, B, H, W, 0, 0, C, KH,
                                         dtype, (hipStream_t)stream);
        if (r != -1) return r;
    }
    if (int e = pdw_dwconv_dgrad(gy, w, dx, B, H, W, C, KH, KW, SH, SW, PH, PW, DH, DW, dtype, stream)) return e;
    return pdw_dwconv_wgrad(x, gy, dw, workspace, workspace_bytes, B, H, W, C, KH, KW, SH, SW, PH, PW, DH, DW, dtype, stream);
}

size_t pdw_static_scratch_bytes(void) { return kStaticScratchBytes; }

int pdw_static_scratch_init(void) {
    void* p = nullptr;
    return static_scratch("pdw_static_scratch_init", &p);
}

int pdw_dwconv_wgrad_static(const void* x, const void* gy, void* dw, int B, int H, int W, int C, int KH, int KW, int SH,
                            int SW, int PH, int PW, int DH, int DW, int dtype, void* stream) {
    if (int e = check_conv("pdw_dwconv_wgrad_static", x, gy, dw, B, H, W, C, KH, KW, SH, SW, PH, PW, DH, DW, dtype))
        return e;
    if (reduce_deferring())
        return set_error("pdw_dwconv_wgrad_static: not available between pdw_reduce_defer_begin and the flush (the "
                         "shared scratch would have to stay untouched until then)"), 1;
    const size_t need = pdw_dwconv_wgrad_workspace_bytes(B, H, W, C, KH, KW, SH, SW, PH, PW, DH, DW, dtype);
    if (need > kStaticScratchBytes)
        return set_error("pdw_dwconv_wgrad_static: these extents need %zu bytes of scratch, the static buffer holds "
                         "%zu; use pdw_dwconv_wgrad with a workspace", need, kStaticScratchBytes), 1;
    void* ws = nullptr;
    if (int e = static_scratch("pdw_dwconv_wgrad_static", &ws)) return e;
    return pdw_dwconv_wgrad(x, gy, dw, ws, kStaticScratchBytes, B, H, W, C, KH, KW, SH, SW, PH, PW, DH, DW, dtype, stream);
}

int pdw_dwconv_wgrad_pair(const void* x0, const void* gy0, void* dw0, void* workspace0, size_t workspace0_bytes, int H0,
                          int W0, const void* x1, const void* gy1, void* dw1, void* workspace1, size_t workspace1_bytes,
                          int H1, int W1, int B, int C, int K, int dtype, void* stream) {
    const int P = K / 2;
    if (int e = check_conv("pdw_dwconv_wgrad_pair", x0, gy0, dw0, B, H0, W0, C, K, K, 1, 1, P, P, 1, 1, dtype)) return e;
    if (int e = check_conv("pdw_dwconv_wgrad_pair", x1, gy1, dw1, B, H1, W1, C, K, K, 1, 1, P, P, 1, 1, dtype)) return e;
    if (!(K & 1)) return set_error("pdw_dwconv_wgrad_pair: odd filter size needed (K=%d)", K), 1;
    if (!dw0 || !dw1) return set_error("pdw_dwconv_wgrad_pair: null dw"), 1;
    const size_t need0 = pdw_dwconv_wgrad_workspace_bytes(B, H0, W0, C, K, K, 1, 1, P, P, 1, 1, dtype);
    const size_t need1 = pdw_dwconv_wgrad_workspace_bytes(B, H1, W1, C, K, K, 1, 1, P, P, 1, 1, dtype);
    if (!workspace0 || workspace0_bytes < need0 || !workspace1 || workspace1_bytes < need1)
        return set_error("pdw_dwconv_wgrad_pair: workspaces of %zu and %zu bytes given, %zu and %zu needed",
                         workspace0_bytes, workspace1_bytes, need0, need1), 1;
    if (B > 0) {
        const int r = dwconv_wgrad_pair_launch(x0, gy0, dw0, workspace0, H0, W0, x1, gy1, dw1, workspace1, H1, W1, B, C,
                                               K, P, P, dtype, (hipStream_t)stream);
        if (r != -1) return r;
    }
    if (int e = pdw_dwconv_wgrad(x0, gy0, dw0, workspace0, workspace0_bytes, B, H0, W0, C, K, K, 1, 1, P, P, 1, 1, dtype,
                                 stream))
        return e;
    return pdw_dwconv_wgrad(x1, gy1, dw1, workspace1, workspace1_bytes, B, H1, W1, C, K, K, 1, 1, P, P, 1, 1, dtype,
                            stream);
}

int pdw_dwconv_bwd3(const void* gy0, const void* w0, const void* gp, void* dx, const void* x0, void* dw0, void* workspace0,
                    size_t workspace0_bytes, const void* x1, const void* gy1, void* dw1, void* workspace1,
                    size_t workspace1_bytes, int B, int H, int W, int C, int K, int dtype, void* stream) {
    const int P = K / 2;
    if (!(K & 1)) return set_error("pdw_dwconv_bwd3: odd filter size needed (K=%d)", K), 1;
    if ((H & 1) || (W & 1)) return set_error("pdw_dwconv_bwd3: even extents needed (H=%d W=%d)", H, W), 1;
    if (int e = check_conv("pdw_dwconv_bwd3", x0, gy0, dw0, B, H, W, C, K, K, 1, 1, P, P, 1, 1, dtype)) return e;
    if (int e = check_conv("pdw_dwconv_bwd3", x1, gy1, dw1, B, H / 2, W / 2, C, K, K, 1, 1, P, P, 1, 1, dtype)) return e;
    if (!w0 || !gp || !dx || !dw0 || !dw1) return set_error("pdw_dwconv_bwd3: null pointer"), 1;
    const size_t need0 = pdw_dwconv_wgrad_workspace_bytes(B, H, W, C, K, K, 1, 1, P, P, 1, 1, dtype);
    const size_t need1 = pdw_dwconv_wgrad_workspace_bytes(B, H / 2, W / 2, C, K, K, 1, 1, P, P, 1, 1, dtype);
    if (!workspace0 || workspace0_bytes < need0 || !workspace1 || workspace1_bytes < need1)
        return set_error("pdw_dwconv_bwd3: workspaces of %zu and %zu bytes given, %zu and %zu needed", workspace0_bytes,
                         workspace1_bytes, need0, need1), 1;
    if (B == 0) return 0;
    const int r = !dwconv_bwd3_covers(B, W, C) ? -1
                                               : dwconv_bwd3_launch(gy0, w0, gp, dx, x0, dw0, workspace0, x1, gy1, dw1, workspace1,
                                                                    B, H, W, H / 2, W / 2, C, K, dtype, (hipStream_t)stream);
    if (r == -1) return set_error("pdw_dwconv_bwd3: case not covered (B=%d H=%d W=%d C=%d K=%d dtype=%d)", B, H, W, C, K, dtype), 3;
    return r;
}

int pdw_dwconv_bwd3_plan(int B, int H, int W, int C, int K, int dtype, int* bands) {
    if (!bands || !valid_dtype(dtype) || B < 1 || H < 2 || W < 2 || C < 1 || K < 1 || !(K & 1) || (H & 1) || (W & 1))
        return set_error("pdw_dwconv_bwd3_plan: bad arguments (B=%d H=%d W=%d C=%d K=%d dtype=%d)", B, H, W, C, K, dtype), 1;
    const int r = !dwconv_bwd3_covers(B, W, C) ? -1
                                               : dwconv_bwd3_launch(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr,
                                                                    nullptr, nullptr, nullptr, B, H, W, H / 2, W / 2, C, K, dtype, nullptr, bands);
    if (r == -1) return set_error("pdw_dwconv_bwd3_plan: case not covered"), 3;
    return r;
}

int pdw_dwconv_fwd2_supported(int B, int H, int W, int C, int K, int dtype) {
    return valid_dtype(dtype) && dwconv_fwd2_covers(B, H, W, C, K, dtype) ? 1 : 0;
}

int pdw_dwconv_fwd2(const void* x0, const void* w0, void* y0, const void* x1, const void* w1, void* y1, int B, int H, int W,
                    int C, int K, int dtype, void* stream) {
    const int P = K / 2;
    if (!(K & 1)) return set_error("pdw_dwconv_fwd2: odd filter size needed (K=%d)", K), 1;
    if ((H & 1) || (W & 1)) return set_error("pdw_dwconv_fwd2: even extents needed (H=%d W=%d)", H, W), 1;
    if (int e = check_conv("pdw_dwconv_fwd2", x0, w0, y0, B, H, W, C, K, K, 1, 1, P, P, 1, 1, dtype)) return e;
    if (int e = check_conv("pdw_dwconv_fwd2", x1, w1, y1, B, H / 2, W / 2, C, K, K, 1, 1, P, P, 1, 1, dtype)) return e;
    if (B == 0) return 0;
    const int r = !dwconv_fwd2_covers(B, H, W, C, K, dtype)
                      ? -1
                      : dwconv_fwd2_launch(x0, w0, y0, x1, w1, y1, B, H, W, H / 2, W / 2, C, K, dtype, (hipStream_t)stream);
    if (r == -1) return set_error("pdw_dwconv_fwd2: case not covered (B=%d H=%d W=%d C=%d K=%d dtype=%d)", B, H, W, C, K, dtype), 3;
    return r;
}

int pdw_dwconv_fwd2_mean(const void* x0, const void* w0, void* y0, int ldy0, int ych0, const void* x1, const void* w1,
                         void* y1, int ldy1, int ych1, int B, int H, int W, int C, int K, const float* parts, int nparts,
                         const void* w_pool, const void* b_pool, const void* b_out, void* m, float* rowbias, int P, int D,
                         int dtype, void* stream) {
    const int Pd = K / 2;
    if (!(K & 1)) return set_error("pdw_dwconv_fwd2_mean: odd filter size needed (K=%d)", K), 1;
    if ((H & 1) || (W & 1)) return set_error("pdw_dwconv_fwd2_mean: even extents needed (H=%d W=%d)", H, W), 1;
    if (int e = check_conv("pdw_dwconv_fwd2_mean", x0, w0, y0, B, H, W, C, K, K, 1, 1, Pd, Pd, 1, 1, dtype)) return e;
    if (int e = check_conv("pdw_dwconv_fwd2_mean", x1, w1, y1, B, H / 2, W / 2, C, K, K, 1, 1, Pd, Pd, 1, 1, dtype)) return e;
    if (B < 1 || P < 1 || D < 1 || nparts < 1)
        return set_error("pdw_dwconv_fwd2_mean: bad extents B=%d P=%d D=%d nparts=%d", B, P, D, nparts), 1;
    if (!parts || !w_pool || !m || !rowbias) return set_error("pdw_dwconv_fwd2_mean: null pointer"), 1;
    if ((ldy0 > 0) != (ldy1 > 0) || ldy0 < 0 || ldy1 < 0 || ych0 < 0 || ych1 < 0 ||
        (ldy0 > 0 && ((C & 1) || ldy0 < ych0 + C / 2 || ldy1 < ych1 + C / 2)))
        return set_error("pdw_dwconv_fwd2_mean: gated stores need even C and ych + C/2 <= ldy for both scales (C=%d ldy=%d,%d "
                         "ych=%d,%d)", C, ldy0, ldy1, ych0, ych1), 1;
    int r = -1;
    if (dwconv_fwd2_covers(B, H, W, C, K, dtype) && pool_branch_v8_ok(w_pool, m, parts, B, D, dtype) && !(reinterpret_cast<uintptr_t>(rowbias) & 15)) {
        const PoolFwdJob job{parts, nparts, B, D, 1.f / (float)P, w_pool, b_pool, b_out, m, rowbias};
        r = dwconv_fwd2_launch(x0, w0, y0, x1, w1, y1, B, H, W, H / 2, W / 2, C, K, dtype, (hipStream_t)stream, ldy0, ych0, ldy1, ych1,
                               &job);
    }
    if (r == -1)
        return set_error("pdw_dwconv_fwd2_mean: case not covered (B=%d H=%d W=%d C=%d K=%d D=%d dtype=%d)", B, H, W, C, K, D,
                         dtype), 3;
    return r;
}

int pdw_dwconv_fwd2_gate(const void* x0, const void* w0, void* y0, int ldy0, int ych0, const void* x1, const void* w1,
                         void* y1, int ldy1, int ych1, int B, int H, int W, int C, int K, int dtype, void* stream) {
    const int P = K / 2;
    if (!(K & 1)) return set_error("pdw_dwconv_fwd2_gate: odd filter size needed (K=%d)", K), 1;
    if ((H & 1) || (W & 1)) return set_error("pdw_dwconv_fwd2_gate: even extents needed (H=%d W=%d)", H, W), 1;
    if (int e = check_conv("pdw_dwconv_fwd2_gate", x0, w0, y0, B, H, W, C, K, K, 1, 1, P, P, 1, 1, dtype)) return e;
    if (int e = check_conv("pdw_dwconv_fwd2_gate", x1, w1, y1, B, H / 2, W / 2, C, K, K, 1, 1, P, P, 1, 1, dtype)) return e;
    if (ldy0 == 0) ldy0 = C / 2;
    if (ldy1 == 0) ldy1 = C / 2;
    if ((C & 1) || ych0 < 0 || ych1 < 0 || ldy0 < ych0 + C / 2 || ldy1 < ych1 + C / 2)
        return set_error("pdw_dwconv_fwd2_gate: need even C and ych + C/2 <= ldy (C=%d ldy=%d,%d ych=%d,%d)", C, ldy0, ldy1,
                         ych0, ych1), 1;
    if (B == 0) return 0;
    const int r = !dwconv_fwd2_covers(B, H, W, C, K, dtype) ? -1
                                                            : dwconv_fwd2_launch(x0, w0, y0, x1, w1, y1, B, H, W, H / 2, W / 2, C, K, dtype,
                                                                                 (hipStream_t)stream, ldy0, ych0, ldy1, ych1);
    if (r == -1)
        return set_error("pdw_dwconv_fwd2_gate: case not covered (B=%d H=%d W=%d C=%d K=%d dtype=%d)", B, H, W, C, K, dtype), 3;
    return r;
}

int pdw_avgpool_fwd(const void* x, void* y, int B, int H, int W, int C, int h, int w, int dtype, void* stream) {
    if (int e = check_resample("pdw_avgpool_fwd", x, y, B, H, W, C, h, w, dtype)) return e;
    return avgpool_fwd_launch(x, y, B, H, W, C, h, w, dtype, (hipStream_t)stream);
}

int pdw_avgpool_bwd(const void* gy, void* gx, int B, int H, int W, int C, int h, int w, int accumulate, int dtype,
                    void* stream) {
    if (int e = check_resample("pdw_avgpool_bwd", gy, gx, B, H, W, C, h, w, dtype)) return e;
    return avgpool_bwd_launch(gy, gx, B, H, W, C, h, w, accumulate ? 1 : 0, dtype, (hipStream_t)stream);
}

int pdw_bilinear_fwd(const void* x, void* y, int B, int h, int w, int C, int H, int W, int ldy, int dtype,
                     void* stream) {
    if (int e = check_resample("pdw_bilinear_fwd", x, y, B, H, W, C, h, w, dtype)) return e;
    if (ldy == 0) ldy = C;
    if (ldy < C) return set_error("pdw_bilinear_fwd: ldy=%d smaller than C=%d", ldy, C), 1;
    return bilinear_fwd_launch(x, y, B, h, w, C, H, W, ldy, dtype, (hipStream_t)stream);
}

int pdw_bilinear_bwd(const void* gy, void* gx, int B, int h, int w, int C, int H, int W, int ldgy, int dtype,
                     void* stream) {
    if (int e = check_resample("pdw_bilinear_bwd", gy, gx, B, H, W, C, h, w, dtype)) return e;
    if (ldgy == 0) ldgy = C;
    if (ldgy < C) return set_error("pdw_bilinear_bwd: ldgy=%d smaller than C=%d", ldgy, C), 1;
    return bilinear_bwd_launch(gy, gx, B, h, w, C, H, W, ldgy, dtype, (hipStream_t)stream);
}

int pdw_gate_fwd(const void* x, void* y, long long M, int I, int ldy, int dtype, void* stream) {
    if (!valid_dtype(dtype)) return set_error("pdw_gate_fwd: unknown dtype %d", dtype), 1;
    if (M < 0 || I < 2 || (I & 1)) return set_error("pdw_gate_fwd: need M >= 0 and even I >= 2 (M=%lld I=%d)", M, I), 1;
    if (M > 0 && (!x || !y)) return set_error("pdw_gate_fwd: null pointer"), 1;
    if (ldy == 0) ldy = I / 2;
    if (ldy < I / 2) return set_error("pdw_gate_fwd: ldy=%d smaller than I/2=%d", ldy, I / 2), 1;
    return gate_fwd_launch(x, y, M, I, ldy, dtype, (hipStream_t)stream);
}

int pdw_gate_bwd(const void* x, const void* gy, void* gx, long long M, int I, int ldgy, int dtype, void* stream) {
    if (!valid_dtype(dtype)) return set_error("pdw_gate_bwd: unknown dtype %d", dtype), 1;
    if (M < 0 || I < 2 || (I & 1)) return set_error("pdw_gate_bwd: need M >= 0 and even I >= 2 (M=%lld I=%d)", M, I), 1;
    if (M > 0 && (!x || !gy || !gx)) return set_error("pdw_gate_bwd: null pointer"), 1;
    if (ldgy == 0) ldgy = I / 2;
    if (ldgy < I / 2) return set_error("pdw_gate_bwd: ldgy=%d smaller than I/2=%d", ldgy, I / 2), 1;
    return gate_bwd_launch(x, gy, gx, M, I, ldgy, dtype, (hipStream_t)stream);
}

int pdw_gate_bilinear_fwd(const void* x, void* y, int B, int h, int w, int I, int H, int W, int ldy, int dtype,
                          void* stream) {
    if (int e = check_resample("pdw_gate_bilinear_fwd", x, y, B, H, W, I, h, w, dtype)) return e;
    if (I < 2 || (I & 1)) return set_error("pdw_gate_bilinear_fwd: need even I >= 2 (I=%d)", I), 1;
    if (ldy == 0) ldy = I / 2;
    if (ldy < I / 2) return set_error("pdw_gate_bilinear_fwd: ldy=%d smaller than I/2=%d", ldy, I / 2), 1;
    return gate_bilinear_fwd_launch(x, y, B, h, w, I, H, W, ldy, dtype, (hipStream_t)stream);
}

int pdw_bilinear_gate_bwd(const void* gy, const void* x, void* gx, int B, int h, int w, int I, int H, int W, int ldgy,
                          int dtype, void* stream) {
    if (int e = check_resample("pdw_bilinear_gate_bwd", gy, gx, B, H, W, I, h, w, dtype)) return e;
    if (I < 2 || (I & 1)) return set_error("pdw_bilinear_gate_bwd: need even I >= 2 (I=%d)", I), 1;
    if (H != 2 * h || W != 2 * w || h < 2 || w < 2)
        return set_error("pdw_bilinear_gate_bwd: needs H = 2h, W = 2w, h,w >= 2 (h=%d w=%d H=%d W=%d); use "
                         "pdw_bilinear_bwd + pdw_gate_bwd", h, w, H, W), 1;
    if ((long long)B * h * w > 0 && !x) return set_error("pdw_bilinear_gate_bwd: null pointer"), 1;
    if (ldgy == 0) ldgy = I / 2;
    if (ldgy < I / 2) return set_error("pdw_bilinear_gate_bwd: ldgy=%d smaller than I/2=%d", ldgy, I / 2), 1;
    return bilinear_gate_bwd_launch(gy, x, gx, B, h, w, I, H, W, ldgy, dtype, (hipStream_t)stream);
}

int pdw_gate_pair_fwd(const void* xf, const void* xh, void* y, int B, int H, int W, int h, int w, int I, int ldy,
                      int dtype, void* stream) {
    if (int e = check_resample("pdw_gate_pair_fwd", xh, y, B, H, W, I, h, w, dtype)) return e;
    if (I < 2 || (I & 1)) return set_error("pdw_gate_pair_fwd: need even I >= 2 (I=%d)", I), 1;
    if (B > 0 && !xf) return set_error("pdw_gate_pair_fwd: null pointer"), 1;
    if (ldy == 0) ldy = I;
    if (ldy < I) return set_error("pdw_gate_pair_fwd: ldy=%d smaller than I=%d", ldy, I), 1;
    return gate_pair_fwd_launch(xf, xh, y, B, H, W, h, w, I, ldy, dtype, (hipStream_t)stream);
}

int pdw_gate_pair_bwd(const void* gy, const void* xf, const void* xh, void* gxf, void* gxh, int B, int H, int W, int h,
                      int w, int I, int ldgy, int dtype, void* stream) {
    if (int e = check_resample("pdw_gate_pair_bwd", gy, gxh, B, H, W, I, h, w, dtype)) return e;
    if (I < 2 || (I & 1)) return set_error("pdw_gate_pair_bwd: need even I >= 2 (I=%d)", I), 1;
    if (B > 0 && (!xf || !xh || !gxf)) return set_error("pdw_gate_pair_bwd: null pointer"), 1;
    if (ldgy == 0) ldgy = I;
    if (ldgy < I) return set_error("pdw_gate_pair_bwd: ldgy=%d smaller than I=%d", ldgy, I), 1;
    const int r = gate_pair_bwd_launch(gy, xf, xh, gxf, gxh, B, H, W, h, w, I, ldgy, dtype, (hipStream_t)stream);
    if (r == -1) return set_error("pdw_gate_pair_bwd: case not covered (B=%d H=%d W=%d h=%d w=%d)", B, H, W, h, w), 3;
    return r;
}

size_t pdw_spatial_sum_workspace_bytes(int B, int P, int C) {
    if (B < 1 || P < 1 || C < 1) return 0;
    return spatial_sum_workspace(B, P, C);
}

int pdw_spatial_sum(const void* x, float* out, void* workspace, size_t workspace_bytes, int B, int P, int C, int dtype,
                    void* stream) {
    if (!valid_dtype(dtype)) return set_error("pdw_spatial_sum: unknown dtype %d", dtype), 1;
    if (B < 0 || P < 1 || C < 1) return set_error("pdw_spatial_sum: bad extents B=%d P=%d C=%d", B, P, C), 1;
    if (B == 0) return 0;
    if (!x || !out) return set_error("pdw_spatial_sum: null pointer"), 1;
    const size_t need = spatial_sum_workspace(B, P, C);
    if (!workspace || workspace_bytes < need)
        return set_error("pdw_spatial_sum: workspace of %zu bytes given, %zu needed", workspace_bytes, need), 1;
    return spatial_sum_launch(x, out, (float*)workspace, B, P, C, dtype, (hipStream_t)stream);
}

int pdw_add_rowbias(void* y, const float* v, int B, int P, int C, int dtype, void* stream) {
    if (!valid_dtype(dtype)) return set_error("pdw_add_rowbias: unknown dtype %d", dtype), 1;
    if (B < 0 || P < 0 || C < 1) return set_error("pdw_add_rowbias: bad extents B=%d P=%d C=%d", B, P, C), 1;
    if (B == 0 || P == 0) return 0;
    if (!y || !v) return set_error("pdw_add_rowbias: null pointer"), 1;
    return add_rowbias_launch(y, v, B, P, C, dtype, (hipStream_t)stream);
}

size_t pdw_pool_branch_workspace_bytes(int B, int P, int D) {
    if (B < 1 || P < 1 || D < 1) return 0;
    return pool_branch_workspace(B, P, D);
}

int pdw_pool_branch_fwd(const void* x, const void* w_pool, const void* b_pool, const void* b_out, void* m,
                        float* rowbias, void* workspace, size_t workspace_bytes, int B, int P, int D, int dtype,
                        void* stream) {
    if (!valid_dtype(dtype)) return set_error("pdw_pool_branch_fwd: unknown dtype %d", dtype), 1;
    if (B < 0 || P < 1 || D < 1) return set_error("pdw_pool_branch_fwd: bad extents B=%d P=%d D=%d", B, P, D), 1;
    if (B == 0) return 0;
    if (!x || !w_pool || !m || !rowbias) return set_error("pdw_pool_branch_fwd: null pointer"), 1;
    if (!workspace || workspace_bytes < pool_branch_workspace(B, P, D))
        return set_error("pdw_pool_branch_fwd: workspace too small"), 1;
    return pool_branch_fwd_launch(x, w_pool, b_pool, b_out, m, rowbias, (float*)workspace, B, P, D, dtype,
                                  (hipStream_t)stream);
}

int pdw_pool_branch_bwd(const void* gy, const void* m, const void* w_pool, void* gbias, void* gbias2, void* gw_pool,
                        float* dmean, void* workspace, size_t workspace_bytes, int B, int P, int D, int dtype,
                        void* stream) {
    if (!valid_dtype(dtype)) return set_error("pdw_pool_branch_bwd: unknown dtype %d", dtype), 1;
    if (B < 1 || P < 1 || D < 1) return set_error("pdw_pool_branch_bwd: bad extents B=%d P=%d D=%d", B, P, D), 1;
    if (!gy || !m || !w_pool || !gbias || !gw_pool || !dmean) return set_error("pdw_pool_branch_bwd: null pointer"), 1;
    if (!workspace || workspace_bytes < pool_branch_workspace(B, P, D))
        return set_error("pdw_pool_branch_bwd: workspace too small"), 1;
    return pool_branch_bwd_launch(gy, m, w_pool, gbias, gbias2, gw_pool, dmean, (float*)workspace, B, P, D, dtype,
                                  (hipStream_t)stream);
}

int pdw_pool_branch_fwd_parts(const float* parts, int nparts, const void* w_pool, const void* b_pool, const void* b_out,
                              void* m, float* rowbias, int B, int P, int D, int dtype, void* stream) {
    if (!valid_dtype(dtype)) return set_error("pdw_pool_branch_fwd_parts: unknown dtype %d", dtype), 1;
    if (B < 1 || P < 1 || D < 1 || nparts < 1)
        return set_error("pdw_pool_branch_fwd_parts: bad extents B=%d P=%d D=%d nparts=%d", B, P, D, nparts), 1;
    if (!parts || !w_pool || !m || !rowbias) return set_error("pdw_pool_branch_fwd_parts: null pointer"), 1;
    return pool_branch_fwd_launch(nullptr, w_pool, b_pool, b_out, m, rowbias, nullptr, B, P, D, dtype,
                                  (hipStream_t)stream, parts, nparts);
}

int pdw_pool_branch_bwd_parts(const float* parts, int nparts, const void* m, const void* w_pool, void* gbias,
                              void* gbias2, void* gw_pool, float* dmean, void* workspace, size_t workspace_bytes, int B,
                              int P, int D, int dtype, void* stream) {
    if (!valid_dtype(dtype)) return set_error("pdw_pool_branch_bwd_parts: unknown dtype %d", dtype), 1;
    if (B < 1 || P < 1 || D < 1 || nparts < 1)
        return set_error("pdw_pool_branch_bwd_parts: bad extents B=%d P=%d D=%d nparts=%d", B, P, D, nparts), 1;
    if (!parts || !m || !w_pool || !gbias || !gw_pool || !dmean)
        return set_error("pdw_pool_branch_bwd_parts: null pointer"), 1;
    if (!workspace || workspace_bytes < pool_branch_workspace(B, P, D))
        return set_error("pdw_pool_branch_bwd_parts: workspace too small"), 1;
    return pool_branch_bwd_launch(nullptr, m, w_pool, gbias, gbias2, gw_pool, dmean, (float*)workspace, B, P, D, dtype,
                                  (hipStream_t)stream, parts, nparts);
}

int pdw_block_mid_infer(const void* xh, void* y, int B, int H, int W, int h, int w, int G, int ldy, const float* parts,
                        int nparts, const void* w_pool, const void* b_pool, const void* b_out, void* m, float* rowbias,
                        int P, int D, int dtype, void* stream) {
    if (int e = check_resample("pdw_block_mid_infer", xh, y, B, H, W, G, h, w, dtype)) return e;
    if (B < 1 || P < 1 || D < 1 || nparts < 1)
        return set_error("pdw_block_mid_infer: bad extents B=%d P=%d D=%d nparts=%d", B, P, D, nparts), 1;
    if (!parts || !w_pool || !m || !rowbias) return set_error("pdw_block_mid_infer: null pointer"), 1;
    if (ldy == 0) ldy = G;
    if (ldy < G) return set_error("pdw_block_mid_infer: ldy=%d smaller than G=%d", ldy, G), 1;
    const int r = bilinear_pool_fwd_launch(xh, y, B, h, w, G, H, W, ldy, parts, nparts, w_pool, b_pool, b_out, m, rowbias,
                                           P, D, dtype, (hipStream_t)stream);
    if (r != -1) return r;
    if (int e = bilinear_fwd_launch(xh, y, B, h, w, G, H, W, ldy, dtype, (hipStream_t)stream)) return e;
    return pool_branch_fwd_launch(nullptr, w_pool, b_pool, b_out, m, rowbias, nullptr, B, P, D, dtype,
                                  (hipStream_t)stream, parts, nparts);
}

int pdw_block_mid_fwd(const void* xf, const void* xh, void* y, int B, int H, int W, int h, int w, int I, int ldy,
                      const float* parts, int nparts, const void* w_pool, const void* b_pool, const void* b_out, void* m,
                      float* rowbias, int P, int D, int dtype, void* stream) {
    if (int e = check_resample("pdw_block_mid_fwd", xh, y, B, H, W, I, h, w, dtype)) return e;
    if (I < 2 || (I & 1)) return set_error("pdw_block_mid_fwd: need even I >= 2 (I=%d)", I), 1;
    if (B < 1 || P < 1 || D < 1 || nparts < 1)
        return set_error("pdw_block_mid_fwd: bad extents B=%d P=%d D=%d nparts=%d", B, P, D, nparts), 1;
    if (!xf || !parts || !w_pool || !m || !rowbias) return set_error("pdw_block_mid_fwd: null pointer"), 1;
    if (ldy == 0) ldy = I;
    if (ldy < I) return set_error("pdw_block_mid_fwd: ldy=%d smaller than I=%d", ldy, I), 1;
    const int r = block_mid_fwd_launch(xf, xh, y, B, H, W, h, w, I, ldy, parts, nparts, w_pool, b_pool, b_out, m,
                                       rowbias, P, D, dtype, (hipStream_t)stream);
    if (r != -1) return r;
    if (int e = gate_pair_fwd_launch(xf, xh, y, B, H, W, h, w, I, ldy, dtype, (hipStream_t)stream)) return e;
    return pool_branch_fwd_launch(nullptr, w_pool, b_pool, b_out, m, rowbias, nullptr, B, P, D, dtype,
                                  (hipStream_t)stream, parts, nparts);
}

int pdw_block_mid_bwd(const void* gy, const void* xf, const void* xh, void* gxf, void* gxh, int B, int H, int W, int h,
                      int w, int I, int ldgy, const float* parts, int nparts, const void* m, const void* w_pool,
                      void* gbias, void* gbias2, void* gw_pool, float* dmean, void* workspace, size_t workspace_bytes,
                      int P, int D, int dtype, void* stream) {
    if (int e = check_resample("pdw_block_mid_bwd", gy, gxh, B, H, W, I, h, w, dtype)) return e;
    if (I < 2 || (I & 1)) return set_error("pdw_block_mid_bwd: need even I >= 2 (I=%d)", I), 1;
    if (B < 1 || P < 1 || D < 1 || nparts < 1)
        return set_error("pdw_block_mid_bwd: bad extents B=%d P=%d D=%d nparts=%d", B, P, D, nparts), 1;
    if (!xf || !xh || !gxf || !parts || !m || !w_pool || !gbias || !gw_pool || !dmean)
        return set_error("pdw_block_mid_bwd: null pointer"), 1;
    if (H != 2 * h || W != 2 * w || h < 2 || w < 2)
        return set_error("pdw_block_mid_bwd: needs H = 2h, W = 2w, h,w >= 2 (h=%d w=%d H=%d W=%d)", h, w, H, W), 1;
    if (!workspace || workspace_bytes < pool_branch_workspace(B, P, D))
        return set_error("pdw_block_mid_bwd: workspace too small"), 1;
    if (ldgy == 0) ldgy = I;
    if (ldgy < I) return set_error("pdw_block_mid_bwd: ldgy=%d smaller than I=%d", ldgy, I), 1;
    const int r = block_mid_bwd_launch(gy, xf, xh, gxf, gxh, B, H, W, h, w, I, ldgy, parts, nparts, m, w_pool, gbias,
                                       gbias2, gw_pool, dmean, (float*)workspace, P, D, dtype, (hipStream_t)stream);
    if (r != -1) return r;
    if (int e = gate_pair_bwd_launch(gy, xf, xh, gxf, gxh, B, H, W, h, w, I, ldgy, dtype, (hipStream_t)stream)) return e;
    return pool_branch_bwd_launch(nullptr, m, w_pool, gbias, gbias2, gw_pool, dmean, (float*)workspace, B, P, D, dtype,
                                  (hipStream_t)stream, parts, nparts);
}

int pdw_dense_colsum_supported(int K, int NO, int dtype) {
    return (dense_colsum_supported(K, NO, dtype) && dense_wgrad_supported(K, NO, dtype)) ? 1 : 0;
}

int pdw_dense_colsum_rows(void) { return dense_colsum_rows(); }

int pdw_dense_fwd_colsum(const void* x, const void* w, int w_kmajor, const void* bias, const float* rowbias, void* y,
                         float* colsum, long long N, int K, int NO, int P, int dtype, void* stream) {
    if (!valid_dtype(dtype)) return set_error("pdw_dense_fwd_colsum: unknown dtype %d", dtype), 1;
    if (N < 0 || K < 1 || NO < 1) return set_error("pdw_dense_fwd_colsum: bad extents N=%lld K=%d NO=%d", N, K, NO), 1;
    if (N > 0 && (!x || !w || !y || !colsum)) return set_error("pdw_dense_fwd_colsum: null pointer"), 1;
    if (rowbias && P < 1) return set_error("pdw_dense_fwd_colsum: rowbias needs P >= 1"), 1;
    const int r = dense_rows_launch(x, w, w_kmajor ? 1 : 0, bias, rowbias, y, N, K, NO, P, dtype, (hipStream_t)stream,
                                    colsum);
    if (r == -1)
        return set_error("pdw_dense_fwd_colsum: K=%d NO=%d dtype=%d not supported (see pdw_dense_colsum_supported)", K,
                         NO, dtype), 3;
    return r;
}

int pdw_dense_fwd_colsum_pool(const void* x, const void* w, const void* bias, void* y, float* colsum, void* pool, int B,
                              int H, int W, int K, int NO, int dtype, void* stream) {
    if (!valid_dtype(dtype)) return set_error("pdw_dense_fwd_colsum_pool: unknown dtype %d", dtype), 1;
    if (B < 0 || H < 2 || W < 2 || (H & 1) || (W & 1) || K < 1 || NO < 1)
        return set_error("pdw_dense_fwd_colsum_pool: bad extents B=%d H=%d W=%d K=%d NO=%d", B, H, W, K, NO), 1;
    if (B > 0 && (!x || !w || !y || !colsum || !pool)) return set_error("pdw_dense_fwd_colsum_pool: null pointer"), 1;
    if (B == 0) return 0;
    const int r = dense_rows_pool_launch(x, w, bias, y, colsum, pool, B, H, W, K, NO, dtype, (hipStream_t)stream);
    if (r == -1)
        return set_error("pdw_dense_fwd_colsum_pool: case not covered (B=%d H=%d W=%d K=%d NO=%d dtype=%d)", B, H, W, K, NO,
                         dtype), 3;
    return r;
}

int pdw_dense_fwd_gated_supported(int H, int W, int I, int D, int dtype) {
    return valid_dtype(dtype) && H > 0 && W > 0 && I > 0 && D > 0 ? dense_mid_rows_supported(H, W, I, D, dtype) : 0;
}

int pdw_dense_fwd_gated(const void* cf, const void* ch, void* cat, const void* w, const void* bias, const float* rowbias,
                        void* y, int B, int H, int W, int I, int D, int ldf, int dtype, void* stream) {
    if (!valid_dtype(dtype)) return set_error("pdw_dense_fwd_gated: unknown dtype %d", dtype), 1;
    if (B < 0 || H < 2 || W < 2 || (H & 1) || (W & 1) || I < 2 || (I & 1) || D < 1)
        return set_error("pdw_dense_fwd_gated: bad extents B=%d H=%d W=%d I=%d D=%d", B, H, W, I, D), 1;
    if (B > 0 && (!cf || !ch || !w || !y)) return set_error("pdw_dense_fwd_gated: null pointer"), 1;
    if (ldf < 0 || (ldf > 0 && (ldf < I / 2 || cat)))
        return set_error("pdw_dense_fwd_gated: gated inputs need ldf >= I/2 and no cat (ldf=%d I=%d)", ldf, I), 1;
    if (B == 0) return 0;
    const int r = dense_mid_rows_launch(cf, ch, cat, w, bias, rowbias, y, B, H, W, I, D, dtype, (hipStream_t)stream, ldf);
    if (r == -1)
        return set_error("pdw_dense_fwd_gated: case not covered (B=%d H=%d W=%d I=%d D=%d dtype=%d)", B, H, W, I, D, dtype), 3;
    return r;
}

int pdw_dense_supported(int K, int NO, int dtype) {
    return (dense_rows_supported(K, NO, dtype) && dense_wgrad_supported(K, NO, dtype)) ? 1 : 0;
}

int pdw_dense_fwd(const void* x, const void* w, int w_kmajor, const void* bias, const float* rowbias, void* y,
                  long long N, int K, int NO, int P, int dtype, void* stream) {
    if (!valid_dtype(dtype)) return set_error("pdw_dense_fwd: unknown dtype %d", dtype), 1;
    if (N < 0 || K < 1 || NO < 1) return set_error("pdw_dense_fwd: bad extents N=%lld K=%d NO=%d", N, K, NO), 1;
    if (N > 0 && (!x || !w || !y)) return set_error("pdw_dense_fwd: null pointer"), 1;
    if (rowbias && P < 1) return set_error("pdw_dense_fwd: rowbias needs P >= 1"), 1;
    const int r = dense_rows_launch(x, w, w_kmajor ? 1 : 0, bias, rowbias, y, N, K, NO, P, dtype, (hipStream_t)stream);
    if (r == -1) return set_error("pdw_dense_fwd: K=%d NO=%d dtype=%d not supported (see pdw_dense_supported)", K, NO, dtype), 3;
    return r;
}

int pdw_dense_fwd_flush(const void* x, const void* w, int w_kmajor, const void* bias, const float* rowbias, void* y,
                        long long N, int K, int NO, int P, int dtype, void* stream) {
    if (!valid_dtype(dtype)) return set_error("pdw_dense_fwd_flush: unknown dtype %d", dtype), 1;
    if (N < 0 || K < 1 || NO < 1) return set_error("pdw_dense_fwd_flush: bad extents N=%lld K=%d NO=%d", N, K, NO), 1;
    if (N > 0 && (!x || !w || !y)) return set_error("pdw_dense_fwd_flush: null pointer"), 1;
    if (rowbias && P < 1) return set_error("pdw_dense_fwd_flush: rowbias needs P >= 1"), 1;
    ReduceJobs jobs;
    const bool ride = N > 0 && dense_rows_supported(K, NO, dtype) && reduce_defer_take(&jobs) > 0;
    const int r = dense_rows_launch(x, w, w_kmajor ? 1 : 0, bias, rowbias, y, N, K, NO, P, dtype, (hipStream_t)stream,
                                    nullptr, ride ? &jobs : nullptr);
    if (r == -1) {
        if (ride) (void)reduce_jobs_launch(jobs, (hipStream_t)stream);  // the reductions still run, on their own
        return set_error("pdw_dense_fwd_flush: K=%d NO=%d dtype=%d not supported (see pdw_dense_supported)", K, NO, dtype), 3;
    }
    return r;
}

size_t pdw_dense_wgrad_workspace_bytes(long long N, int M, int NO) {
    if (N < 0 || M < 1 || NO < 1) return 0;
    return dense_wgrad_workspace(N, M, NO);
}

int pdw_dense_wgrad(const void* a, const void* b, void* dw, void* workspace, size_t workspace_bytes, long long N, int M,
                    int NO, int dtype, void* stream) {
    if (!valid_dtype(dtype)) return set_error("pdw_dense_wgrad: unknown dtype %d", dtype), 1;
    if (N < 0 || M < 1 || NO < 1) return set_error("pdw_dense_wgrad: bad extents N=%lld M=%d NO=%d", N, M, NO), 1;
    if (!dw || (N > 0 && (!a || !b))) return set_error("pdw_dense_wgrad: null pointer"), 1;
    const size_t need = dense_wgrad_workspace(N, M, NO);
    if (!workspace || workspace_bytes < need)
        return set_error("pdw_dense_wgrad: workspace of %zu bytes given, %zu needed", workspace_bytes, need), 1;
    const int r = dense_wgrad_launch(a, b, dw, workspace, N, M, NO, dtype, (hipStream_t)stream);
    if (r == -1) return set_error("pdw_dense_wgrad: M=%d NO=%d dtype=%d not supported", M, NO, dtype), 3;
    return r;
}

int pdw_dense_bwd_pair_supported(int O, int I, int dtype) {
    return valid_dtype(dtype) ? dense_bwd_pair_supported(O, I, dtype) : 0;
}

int pdw_dense_bwd_pair_colsum_supported(int O, int I, int dtype) {
    return valid_dtype(dtype) ? dense_bwd_pair_colsum_supported(O, I, dtype) : 0;
}

int pdw_dense_bwd_pair(const void* gy, const void* w, const void* x, void* dx, float* colsum, void* dw, void* workspace,
                       size_t workspace_bytes, const float* rowbias, int P, long long N, int O, int I, int dtype,
                       void* stream) {
    if (!valid_dtype(dtype)) return set_error("pdw_dense_bwd_pair: unknown dtype %d", dtype), 1;
    if (N < 1 || O < 1 || I < 1) return set_error("pdw_dense_bwd_pair: bad extents N=%lld O=%d I=%d", N, O, I), 1;
    if (!gy || !w || !x || !dx || !dw) return set_error("pdw_dense_bwd_pair: null pointer"), 1;
    const size_t need = dense_wgrad_workspace(N, O, I);
    if (!workspace || workspace_bytes < need)
        return set_error("pdw_dense_bwd_pair: workspace of %zu bytes given, %zu needed", workspace_bytes, need), 1;
    if (rowbias && P < 1) return set_error("pdw_dense_bwd_pair: rowbias needs P >= 1"), 1;
    const int r = dense_bwd_pair_launch(gy, w, x, dx, colsum, dw, workspace, rowbias, P, N, O, I, dtype,
                                        (hipStream_t)stream);
    if (r == -1)
        return set_error("pdw_dense_bwd_pair: O=%d I=%d dtype=%d (P=%d) not covered (see pdw_dense_bwd_pair_supported)",
                         O, I, dtype, P), 3;
    return r;
}

int pdw_norm_fwd(const void* x, const void* weight, const void* bias, void* y, float* stats, long long N, int C, int kind,
                 float eps, int dtype, void* stream) {
    if (int e = check_rows("pdw_norm_fwd", N, C, kind, kNormNone, kActNone, dtype)) return e;
    if (kind == kNormNone) return set_error("pdw_norm_fwd: no norm asked for"), 1;
    if (N > 0 && (!x || !y)) return set_error("pdw_norm_fwd: null pointer"), 1;
    RowArgs p{};
    p.x = x, p.w2 = weight, p.b2 = bias, p.next = y, p.st2 = stats, p.N = N, p.P = N, p.C = C, p.kind2 = kind, p.eps = eps;
    return rows_forward_launch(p, dtype, (hipStream_t)stream);
}

size_t pdw_norm_bwd_workspace_bytes(long long N, int C, int dtype) {
    if (check_rows("pdw_norm_bwd_workspace_bytes", N, C, 0, 0, 0, dtype)) return 0;
    return rows_backward_workspace(N, 1, C, 2, dtype);
}

int pdw_norm_bwd(const void* gy, const void* x, const void* weight, const float* stats, void* gx, void* gweight, void* gbias,
                 void* workspace, size_t workspace_bytes, long long N, int C, int kind, int dtype, void* stream) {
    if (int e = check_rows("pdw_norm_bwd", N, C, kind, kNormNone, kActNone, dtype)) return e;
    if (kind == kNormNone) return set_error("pdw_norm_bwd: no norm asked for"), 1;
    if (N > 0 && (!gy || !x || !stats)) return set_error("pdw_norm_bwd: null pointer"), 1;
    RowArgs p{};
    p.x = x, p.gz = gy, p.w2 = weight, p.st2 = const_cast<float*>(stats), p.gx = gx, p.N = N, p.P = N, p.C = C, p.kind2 = kind;
    return rows_backward_launch(p, nullptr, nullptr, nullptr, gweight, gbias, workspace, workspace_bytes, dtype, (hipStream_t)stream);
}

int pdw_residual_fwd(const void* x, const void* y, const void* gate, const void* scale, const void* weight, const void* bias,
                     const void* next_weight, const void* next_bias, void* out, void* next, float* stats, float* next_stats,
                     long long N, int C, long long P, long long ldgate, int act, int kind, int next_kind, float eps, int dtype,
                     void* stream) {
    if (int e = check_rows("pdw_residual_fwd", N, C, kind, next_kind, act, dtype)) return e;
    if (int e = check_gate("pdw_residual_fwd", gate, N, C, P, &ldgate)) return e;
    if (N > 0 && (!x || !y || !out || (next_kind != kNormNone && !next))) return set_error("pdw_residual_fwd: null pointer"), 1;
    RowArgs p{};
    p.x = x, p.y = y, p.gate = gate, p.scale = scale, p.w = weight, p.b = bias, p.w2 = next_weight, p.b2 = next_bias;
    p.out = out, p.next = next, p.st = stats, p.st2 = next_stats, p.N = N, p.P = P, p.ldg = ldgate, p.C = C;
    p.act = act, p.kind = kind, p.kind2 = next_kind, p.gate_rows = !gate ? 0 : P == 1 ? 2 : 1, p.eps = eps;
    return rows_forward_launch(p, dtype, (hipStream_t)stream);
}

size_t pdw_residual_bwd_workspace_bytes(long long N, int C, long long P, int next_kind, int dtype) {
    if (check_rows("pdw_residual_bwd_workspace_bytes", N, C, 0, next_kind, 0, dtype)) return 0;
    // (P only where a gate row serves several rows; otherwise all rows are one image)
    return rows_backward_workspace(N, P > 1 && N % P == 0 ? N / P : 1, C, next_kind == kNormNone ? 2 : 4, dtype);
}

int pdw_residual_bwd(const void* gout, const void* gnext, const void* x, const void* y, const void* gate, const void* scale,
                     const void* weight, const void* bias, const void* next_weight, const float* stats, const float* next_stats,
                     void* gx, void* gy, void* ggate, void* gscale, void* gweight, void* gbias, void* gnext_weight,
                     void* gnext_bias, void* workspace, size_t workspace_bytes, long long N, int C, long long P,
                     long long ldgate, int act, int kind, int next_kind, int dtype, void* stream) {
    if (int e = check_rows("pdw_residual_bwd", N, C, kind, next_kind, act, dtype)) return e;
    if (int e = check_gate("pdw_residual_bwd", gate, N, C, P, &ldgate)) return e;
    const bool next = next_kind != kNormNone;
    if (N > 0 && (!gout || !y || (kind != kNormNone && !stats) || (next && (!gnext || !x || !next_stats)) || (!gate && ggate)))
        return set_error("pdw_residual_bwd: null pointer"), 1;
    RowArgs p{};
    p.go = gout, p.gz = gnext, p.x = x, p.y = y, p.gate = gate, p.scale = scale, p.w = weight, p.b = bias, p.w2 = next_weight;
    p.st = const_cast<float*>(stats), p.st2 = const_cast<float*>(next_stats), p.gx = next ? gx : nullptr, p.gy = gy, p.ggate = ggate;
    p.N = N, p.P = P, p.ldg = ldgate, p.C = C, p.act = act, p.kind = kind, p.kind2 = next_kind;
    p.gate_rows = !gate ? 0 : P == 1 ? 2 : 1;
    return rows_backward_launch(p, gscale, gweight, gbias, gnext_weight, gnext_bias, workspace, workspace_bytes, dtype,
                                (hipStream_t)stream);
}

size_t pdw_scan_states_bytes(int O, long long T, int W, int I) {
    return O < 1 || T < 1 || W < 1 || I < 1 ? 0 : scan_states_bytes((long long)O * W, T, I);
}

size_t pdw_scan_workspace_bytes(int O, long long T, int W, int I, int backward) {
    return O < 1 || T < 1 || W < 1 || I < 1 ? 0 : scan_workspace((long long)O * W, T, I, backward != 0);
}

static ScanStrides strides_of(const long long* s) { return s ? ScanStrides{s[0], s[1], s[2]} : ScanStrides{0, 0, 0}; }

int pdw_scan_fwd(const void* x, const void* g, const float* h0, const int* lengths, void* y, float* last, float* states,
                 void* workspace, size_t workspace_bytes, int O, long long T, int W, int I, const long long* xs,
                 const long long* gs, int reverse, int dtype, void* stream) {
    if (int e = check_scan("pdw_scan_fwd", x, g, xs, gs, O, T, W, I, dtype)) return e;
    if (O == 0 || W == 0 || I == 0) return 0;
    if (T > 0 && !y) return set_error("pdw_scan_fwd: null pointer"), 1;
    ScanArgs p{};
    p.x = x, p.g = g, p.h0 = h0, p.lengths = lengths, p.y = y, p.last = last, p.states = states;
    p.rows = O * W, p.T = T, p.W = W, p.I = I, p.xs = strides_of(xs), p.gs = strides_of(gs), p.reverse = reverse != 0;
    p.dense = {T * W * I, (long long)W * I, I};
    return scan_run(p, false, workspace, workspace_bytes, dtype, (hipStream_t)stream);
}

int pdw_scan_bwd(const void* gy, const float* glast, const void* x, const void* g, const int* lengths, const float* states,
                 void* gx, void* gg, float* gh0, void* workspace, size_t workspace_bytes, int O, long long T, int W, int I,
                 const long long* xs, const long long* gs, const long long* gxs, const long long* ggs, int reverse, int dtype,
                 void* stream) {
    if (int e = check_scan("pdw_scan_bwd", x, g, xs, gs, O, T, W, I, dtype)) return e;
    if (O == 0 || W == 0 || I == 0) return 0;
    if (T > 0 && (!states || (gx && !gxs) || (gg && !ggs))) return set_error("pdw_scan_bwd: null pointer"), 1;
    ScanArgs p{};
    p.x = x, p.g = g, p.gy = gy, p.glast = glast, p.lengths = lengths, p.states = const_cast<float*>(states);
    p.gx = gx, p.gg = gg, p.gh0 = gh0, p.rows = O * W, p.T = T, p.W = W, p.I = I, p.reverse = reverse != 0;
    p.xs = strides_of(xs), p.gs = strides_of(gs), p.gxs = strides_of(gxs), p.ggs = strides_of(ggs);
    p.dense = {T * W * I, (long long)W * I, I};
    return scan_run(p, true, workspace, workspace_bytes, dtype, (hipStream_t)stream);
}

int pdw_scan_step(const void* x, const void* g, const float* state, float* new_state, void* y, long long B, int C,
                  long long ldx, long long ldg, int dtype, void* stream) {
    if (!valid_dtype(dtype)) return set_error("pdw_scan_step: unknown dtype %d", dtype), 1;
    if (B < 0 || C < 0) return set_error("pdw_scan_step: bad extents B=%lld C=%d", B, C), 1;
    if (B == 0 || C == 0) return 0;
    if (!x || !g || !state || !new_state || !y) return set_error("pdw_scan_step: null pointer"), 1;
    return scan_step_launch(x, g, state, new_state, y, B, C, ldx, ldg, dtype, (hipStream_t)stream);
}

static int rotary_args(const char* fn, const pdw_rotary* c, RotaryArgs& p) {
    if (!c) return set_error("%s: null pointer", fn), 1;
    if (!valid_dtype(c->dtype)) return set_error("%s: unknown dtype %d", fn, c->dtype), 1;
    if (c->kind < kRotaryNone || c->kind > kRotaryL2 || c->position_type < kPositionGrid || c->position_type > kPositionF32)
        return set_error("%s: unknown kind %d or type of positions %d", fn, c->kind, c->position_type), 1;
    if (c->d < 1 || c->d > kRotaryMaxDim || c->axes < 1 || c->axes > 3 || c->tokens < 0 || c->heads[0] < 0 || c->heads[1] < 0)
        return set_error("%s: bad extents d=%d axes=%d tokens=%lld heads=%d,%d", fn, c->d, c->axes, c->tokens, c->heads[0], c->heads[1]), 1;
    // (a workgroup counts the rows of its tokens in 32 bits)
    if (c->heads[0] > 1 << 16 || c->heads[1] > 1 << 16) return set_error("%s: more than 65536 heads", fn), 1;
    int P = 0;
    for (int a = 0; a < c->axes; ++a) {
        if (c->sections[a] < 0 || c->sections[a] > kRotaryMaxDim) return set_error("%s: section %d of %d pairs", fn, a, c->sections[a]), 1;
        P += c->sections[a], p.ends[a] = P;
    }
    for (int a = c->axes; a < 3; ++a) p.ends[a] = P;
    if (2 * P > c->d) return set_error("%s: %d pairs of %d channels", fn, P, c->d), 1;
    if (c->kind == kRotaryNone && (c->weight[0] || c->weight[1])) return set_error("%s: weight without a norm", fn), 1;
    if (c->tokens > 0 && ((c->heads[0] && !c->x[0]) || (c->heads[1] && !c->x[1]))) return set_error("%s: null pointer", fn), 1;
    p.grid[0] = p.grid[1] = p.grid[2] = 1;
    if (c->position_type == kPositionGrid) {
        for (int a = 0; a < c->axes; ++a) {
            if (c->tokens > 0 && c->grid[a] < 1) return set_error("%s: grid extent %d", fn, c->grid[a]), 1;
            p.grid[3 - c->axes + a] = c->grid[a] < 1 ? 1 : c->grid[a];
        }
    } else if (c->tokens > 0 && (!c->positions || c->positions_rows < 1)) {
        return set_error("%s: no positions", fn), 1;
    }
    for (int s = 0; s < 2; ++s)
        p.x[s] = c->x[s], p.xt[s] = c->xt[s], p.xh[s] = c->xh[s], p.heads[s] = c->heads[s], p.w[s] = c->weight[s];
    p.positions = c->positions, p.frequencies = c->frequencies, p.N = c->tokens, p.np = c->positions_rows, p.d = c->d, p.P = P;
    p.axes = c->axes, p.kind = c->kind, p.neighbours = c->neighbours != 0, p.pkind = c->position_type, p.eps = c->eps;
    if (!c->frequencies) {
        int i = 0;
        for (int a = 0; a < c->axes; ++a)
            for (int j = 0; j < c->sections[a]; ++j) p.turns[i++] = std::pow(c->base, -(double)j / c->sections[a]) * 0.15915494309189535;
    }
    return 0;
}

int pdw_rotary_fwd(const pdw_rotary* c, void* const y[2], void* stream) {
    RotaryArgs p{};
    if (int e = rotary_args("pdw_rotary_fwd", c, p)) return e;
    if (p.N == 0 || (!p.heads[0] && !p.heads[1])) return 0;
    if (!y || (p.heads[0] && !y[0]) || (p.heads[1] && !y[1])) return set_error("pdw_rotary_fwd: null pointer"), 1;
    p.y[0] = y[0], p.y[1] = y[1];
    return rotary_run(p, false, nullptr, nullptr, nullptr, 0, c->dtype, (hipStream_t)stream);
}

size_t pdw_rotary_bwd_workspace_bytes(int d) { return d < 1 || d > kRotaryMaxDim ? 0 : rotary_workspace(d); }

int pdw_rotary_bwd(const pdw_rotary* c, const void* const gy[2], void* const gx[2], void* const gweight[2], void* workspace,
                   size_t workspace_bytes, void* stream) {
    RotaryArgs p{};
    if (int e = rotary_args("pdw_rotary_bwd", c, p)) return e;
    if (c->kind == kRotaryNone && gweight && (gweight[0] || gweight[1])) return set_error("pdw_rotary_bwd: gradient of a weight without a norm"), 1;
    if (p.N == 0 || (!p.heads[0] && !p.heads[1]))
        return gweight ? rotary_no_rows(gweight[0], gweight[1], p.d, c->dtype, (hipStream_t)stream) : 0;
    if (!gy || !gx || !gweight || (p.heads[0] && !gy[0]) || (p.heads[1] && !gy[1])) return set_error("pdw_rotary_bwd: null pointer"), 1;
    for (int s = 0; s < 2; ++s) p.gy[s] = gy[s], p.y[s] = gx[s];
    return rotary_run(p, true, gweight[0], gweight[1], workspace, workspace_bytes, c->dtype, (hipStream_t)stream);
}

static int delta_args(const char* fn, const pdw_delta* c, DeltaArgs& p) {
    if (!c) return set_error("%s: null pointer", fn), 1;
    if (!valid_dtype(c->dtype)) return set_error("%s: unknown dtype %d", fn, c->dtype), 1;
    if (c->O < 0 || c->W < 0 || c->T < 0 || c->T > 0x7fffffffLL - kDeltaChunk || c->Hk < 0 || c->Hv < 0)
        return set_error("%s: bad extents O=%d T=%lld W=%d heads=%d,%d", fn, c->O, c->T, c->W, c->Hk, c->Hv), 1;
    if (c->dk < 1 || c->dk > PDW_DELTA_MAX_CHANNELS || c->dv < 1 || c->dv > PDW_DELTA_MAX_CHANNELS)
        return set_error("%s: %d and %d channels of a head, 1 to %d are possible", fn, c->dk, c->dv, PDW_DELTA_MAX_CHANNELS), 1;
    if (c->Hv ? c->Hk < 1 || c->Hv % c->Hk : c->Hk) return set_error("%s: %d value heads for %d key heads", fn, c->Hv, c->Hk), 1;
    const long long rows = (long long)c->O * c->W;
    if (rows > 0x7fffffffLL || rows * c->Hv > 0x7fffffffLL) return set_error("%s: more than 2^31 - 1 chains", fn), 1;
    if (rows * c->Hv && c->T && (!c->q || !c->k || !c->v || !c->g || !c->b)) return set_error("%s: null pointer", fn), 1;
    auto strides = [](const long long* s) { return DeltaStrides{s[0], s[1], s[2], s[3]}; };
    p.q = c->q, p.k = c->k, p.v = c->v, p.g = c->g, p.b = c->b;
    p.qs = strides(c->qs), p.ks = strides(c->ks), p.vs = strides(c->vs), p.gs = strides(c->gs), p.bs = strides(c->bs);
    auto dense = [&](long long H, long long d) { return DeltaStrides{c->T * c->W * H * d, c->W * H * d, H * d, d}; };
    p.ys = dense(c->Hv, c->dv), p.gqs = dense(c->Hk, c->dk), p.gvs = p.ys, p.ggs = dense(c->Hv, 1);
    p.h0 = c->h0, p.lengths = c->lengths, p.T = (int)c->T, p.O = c->O, p.W = c->W, p.Hk = c->Hk, p.Hv = c->Hv, p.dk = c->dk, p.dv = c->dv;
    p.chains = (int)(rows * c->Hv), p.reverse = c->reverse != 0, p.logits = c->logits != 0, p.gates_f32 = c->gates_f32 != 0, p.scale = c->scale;
    return 0;
}

size_t pdw_delta_states_bytes(const pdw_delta* c) {
    DeltaArgs p{};
    return delta_args("pdw_delta_states_bytes", c, p) ? 0 : delta_states_bytes(p.chains, p.T, p.dk, p.dv, c->dtype);
}

size_t pdw_delta_workspace_bytes(const pdw_delta* c, int backward, int with_states) {
    DeltaArgs p{};
    return delta_args("pdw_delta_workspace_bytes", c, p) ? 0 : delta_workspace(p.chains, p.T, p.dk, p.dv, backward != 0, with_states != 0, c->dtype);
}

int pdw_delta_fwd(const pdw_delta* c, void* y, float* last, void* states, void* workspace, size_t workspace_bytes, void* stream) {
    DeltaArgs p{};
    if (int e = delta_args("pdw_delta_fwd", c, p)) return e;
    if (!p.chains) return 0;
    if (p.T && !y) return set_error("pdw_delta_fwd: null pointer"), 1;
    p.y = y, p.last = last;
    return delta_run(p, states, false, workspace, workspace_bytes, c->dtype, (hipStream_t)stream);
}

int pdw_delta_bwd(const pdw_delta* c, const void* gy, const float* glast, const void* states, void* gq, void* gk, void* gv, void* gg,
                  void* gb, float* gh0, void* workspace, size_t workspace_bytes, void* stream) {
    DeltaArgs p{};
    if (int e = delta_args("pdw_delta_bwd", c, p)) return e;
    if (!p.chains) return 0;
    if (p.T && (!gy || !states)) return set_error("pdw_delta_bwd: null pointer"), 1;
    p.gy = gy, p.glast = glast, p.gq = gq, p.gk = gk, p.gv = gv, p.gg = gg, p.gb = gb, p.gh0 = gh0;
    return delta_run(p, const_cast<void*>(states), true, workspace, workspace_bytes, c->dtype, (hipStream_t)stream);
}

int pdw_delta_step(const pdw_delta* c, void* y, float* last, void* stream) {
    DeltaArgs p{};
    if (int e = delta_args("pdw_delta_step", c, p)) return e;
    if (!p.chains) return 0;
    if (!last || (p.T && !y)) return set_error("pdw_delta_step: null pointer"), 1;
    p.y = y, p.last = last;
    return delta_steps_run(p, c->dtype, (hipStream_t)stream);
}

}  // extern "C"
