/*
 * pdw.h - C ABI of libpdw.so: hand-written gfx950 (MI355X) kernels for the pyramid
 * depthwise-convolution block.
 *
 * The reference (IrisRainbowNeko/PyramidConvBlock) has no FFI: its device code is reached
 * through Triton's `kernel[grid](...)` launches inside Python autograd Functions.  Each
 * entry point below replaces one such launch site (cited per function, paths relative to
 * the reference tree) and is what a binding for that site would call.
 *
 * Conventions
 *   - All tensors are dense channels-last: x[B][H][W][C] with C fastest; depthwise
 *     weights are w[KH][KW][C]  (dwconv_triton.py:413-416).
 *   - Every pointer is a DEVICE pointer borrowed for the duration of the call; nothing is
 *     allocated, freed or synchronised inside the library.  Work is enqueued on `stream`
 *     (a hipStream_t passed as void*; NULL = the null stream) of the current device.
 *   - `dtype` is one of PDW_F32 / PDW_F16 / PDW_BF16 and applies to every tensor of the
 *     call.  Arithmetic is fp32 (bf16/fp16 products are exact in fp32), one rounding on store.
 *   - Return value: 0 on success; non-zero on invalid arguments or a failed launch, with a
 *     message available from pdw_last_error() (thread-local).
 *   - Callable from several host threads at once.  The library keeps four pieces of state: the per-thread
 *     error text, the per-thread list of summations recorded between pdw_reduce_defer_begin() and
 *     pdw_reduce_defer_flush(), a once-per-process set-up of each large kernel's LDS limit (guarded by
 *     std::call_once), and bounded caches of launch plans per shape (of the shared launches, the 16-bit matrix-core convolutions and
 *     the vector-ALU kernels with their workspace queries; each behind a mutex and emptied when it reaches 256 shapes; a plan is a
 *     function of the shape alone, so they change no result).  The no-allocation entry point
 *     has a device buffer of its own, described there.  The library reads no environment variables: every launch plan
 *     is a function of the arguments.
 *   - Non-finite inputs: the matrix-core convolution kernels multiply a window of input pixels somewhat larger
 *     than the filter by zero-padded filter operands, so an Inf or NaN input pixel can turn outputs up to
 *     PDW_NONFINITE_REACH pixels beyond the filter's own footprint into NaN (0 * Inf).  Outputs further away, those of
 *     the batch's other images, and all outputs for finite inputs, are unaffected.  The reference masks its loads (dwconv_triton.py:55-86), so
 *     there the value reaches the footprint only.
 */
#ifndef PDW_H_
#define PDW_H_

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { PDW_F32 = 0, PDW_F16 = 1, PDW_BF16 = 2 };

/* See "Non-finite inputs" above: extra pixels, in every direction, by which a non-finite input value can reach
 * beyond the K x K footprint of the filter. */
#define PDW_NONFINITE_REACH 16

/* ABI version of the library (bumped when a signature changes). */
int pdw_version(void);
/* Text of the last error raised on the calling thread ("" if none). */
const char *pdw_last_error(void);

/* Output extent of a convolution axis: (in + 2p - d(k-1) - 1)/s + 1, 0 if empty.
 * dwconv_triton.py:311-312. */
int pdw_conv_out_size(int in, int k, int stride, int pad, int dil);

/* Depthwise cross-correlation  y[b,i,j,c] = sum_{kh,kw} x[b, i*sh-ph+kh*dh, j*sw-pw+kw*dw, c] * w[kh,kw,c],
 * zero outside the image.  x[B,H,W,C] -> y[B,OH,OW,C].
 * Replaces the launch of _depthwise_conv_kernel_optimized, dwconv_triton.py:325-333 (kernel :20-104). */
int pdw_dwconv_fwd(const void *x, const void *w, void *y, int B, int H, int W, int C, int KH, int KW,
                   int SH, int SW, int PH, int PW, int DH, int DW, int dtype, void *stream);

/* pdw_dwconv_fwd plus the adaptive average pool of the same input to (h, wp): y = conv(x), xp[B,h,wp,C] = pool(x).
 * ConvBlock feeds one tensor to the full-resolution conv and, pooled, to the next scale (conv_block.py:14-16, 41);
 * when the pool halves both extents exactly (and the conv keeps them: stride 1, 2*pad = k-1, pad even, 16-bit
 * types, C % 8 == 0) the conv kernel writes the pooled tensor from its staged input window, otherwise
 * pdw_dwconv_fwd and pdw_avgpool_fwd run one after the other. */
int pdw_dwconv_fwd_pool(const void *x, const void *w, void *y, void *xp, int B, int H, int W, int C, int KH, int KW,
                        int SH, int SW, int PH, int PW, int DH, int DW, int h, int wp, int dtype, void *stream);

/* Inference form of SimpleGate's convolution and gate (conv_block.py:17-19) for stride 1 and a square filter:
 *   y[b,i,j, ych + c] = conv(x)[b,i,j,c] * conv(x)[b,i,j,C/2 + c] * sqrt(C/2),   c < C/2,
 * written with a pixel stride of ldy channels (0: C/2), e.g. straight into its slice of the concatenation of
 * conv_block.py:43, so that the convolution output itself never reaches HBM.  The product is formed from the rounded
 * convolution outputs in fp32 and rounded once, as pdw_gate_fwd does.  xp (may be NULL): the 2x2 average pool of x,
 * [B,H/2,W/2,C] (needs even H, W, pad and 2*pad = K-1).  Returns 3 when the fused kernel does not cover the case
 * (it needs a 16-bit dtype, C % 16 == 0, odd K <= 17, ldy and ych multiples of 8, and K <= 13 when xp is asked for): the
 * caller then runs pdw_dwconv_fwd
 * (or pdw_dwconv_fwd_pool) and pdw_gate_fwd.  No counterpart in the reference, which keeps the convolution output for
 * its backward. */
int pdw_dwconv_fwd_gate(const void *x, const void *w, void *y, void *xp, int B, int H, int W, int C, int K, int pad,
                        int ldy, int ych, int dtype, void *stream);

/* Input gradient (exact adjoint of pdw_dwconv_fwd in x): gy[B,OH,OW,C] -> dx[B,H,W,C]; H,W are
 * the forward INPUT extents.  Fully overwrites dx (no pre-zeroing needed).
 * Replaces the launch of _depthwise_conv_backward_input_kernel, dwconv_triton.py:358-366
 * (kernel :119-203), which is only correct for stride 1 and 2*pad == dil*(k-1); this entry
 * point is correct for every stride/pad/dilation. */
int pdw_dwconv_dgrad(const void *gy, const void *w, void *dx, int B, int H, int W, int C, int KH, int KW,
                     int SH, int SW, int PH, int PW, int DH, int DW, int dtype, void *stream);

/* pdw_dwconv_dgrad plus the gradient of an adaptive average pool taken of the same tensor:
 * dx[B,H,W,C] = dgrad(gy) + avgpool_bwd(gp[B,h,wp,C] -> (H,W)).  This is the sum autograd forms for the
 * tensor that feeds both the full-resolution gate and, through conv_block.py:14, a pooled one
 * (conv_block.py:41).  One kernel when the pool halves both extents exactly (stride 1, dilation 1, 16-bit
 * types, C % 8 == 0), otherwise pdw_dwconv_dgrad followed by an accumulating pdw_avgpool_bwd; either way dx is
 * rounded to the storage type after each of the two terms. */
int pdw_dwconv_dgrad_addpool(const void *gy, const void *w, const void *gp, void *dx, int B, int H, int W, int C,
                             int KH, int KW, int SH, int SW, int PH, int PW, int DH, int DW, int h, int wp,
                             int dtype, void *stream);

/* The weight-gradient entry points (pdw_dwconv_wgrad, pdw_dense_wgrad) end with a small kernel that sums their
 * fp32 partial results.  Between pdw_reduce_defer_begin() and pdw_reduce_defer_flush(stream), on the calling host
 * thread, that last step is only recorded (up to 8 of them, further ones run at once as usual), and the flush
 * runs all recorded ones in a single launch on `stream`: the outputs are not valid, and the workspaces must not
 * be reused or freed, until then.  Two entry points take recorded work along in spare workgroups of their own
 * launch, after which the list is empty again: pdw_dense_wgrad (what was recorded before it; its own summation is
 * recorded afterwards) and pdw_dense_fwd_flush below.  pdw_block_mid_bwd records the gradients of the pooled
 * layer's weight and bias (gw_pool, gbias, gbias2) in the same way instead of computing them in its own launch.
 * No counterpart in the reference (its backward launches every kernel separately, dwconv_triton.py:358-385);
 * the ConvBlock backward (conv_block.py:36-49 under autograd) uses it for its weight gradients. */
/* out[i] = sum over p < nparts of parts[p * n + i], added in fp32 in a fixed order and rounded once to `dtype`: the
 * last step of every weight gradient here, on its own for callers that make the partial products themselves (the
 * operator's weight gradient of conv_up / conv_out for widths the dense kernels do not cover is a batched library
 * product over row slabs; autograd of conv_block.py:37, 44).  Subject to the deferral below like the others. */
int pdw_sum_parts(const float *parts, void *out, int nparts, long long n, int dtype, void *stream);
int pdw_reduce_defer_begin(void);
int pdw_reduce_defer_flush(void *stream);
/* pdw_dense_fwd that also runs the reductions recorded so far (see above) in spare workgroups of its own launch;
 * the later pdw_reduce_defer_flush then launches nothing.  For a dense layer that runs after the last kernel that
 * produced the partial results: the input gradient of conv_up at the end of the block's backward. */
int pdw_dense_fwd_flush(const void *x, const void *w, int w_kmajor, const void *bias, const float *rowbias, void *y,
                        long long N, int K, int NO, int P, int dtype, void *stream);

/* Bytes of device scratch pdw_dwconv_wgrad needs for these extents (fp32 partial sums). */
size_t pdw_dwconv_wgrad_workspace_bytes(int B, int H, int W, int C, int KH, int KW, int SH, int SW,
                                        int PH, int PW, int DH, int DW, int dtype);

/* Weight gradient dw[kh,kw,c] = sum_{b,i,j} gy[b,i,j,c] * x[b, i*sh-ph+kh*dh, j*sw-pw+kw*dw, c].
 * Two deterministic passes (per-block fp32 partials in `workspace`, then a fixed-order sum);
 * no atomics, so results are bit-reproducible.  Fully overwrites dw.
 * Replaces the launch of _depthwise_conv_weight_grad_kernel, dwconv_triton.py:377-385
 * (kernel :219-296). */
int pdw_dwconv_wgrad(const void *x, const void *gy, void *dw, void *workspace, size_t workspace_bytes,
                     int B, int H, int W, int C, int KH, int KW, int SH, int SW, int PH, int PW, int DH,
                     int DW, int dtype, void *stream);

/* pdw_dwconv_dgrad and pdw_dwconv_wgrad of one convolution as one call (dwconv_triton.py:334-387): dx from gy and w, dw from x and gy,
 * workspace as for pdw_dwconv_wgrad.  16-bit types with an odd square filter up to 17, stride 1 and padding K/2 run as one launch
 * where that is estimated to end sooner, everything else as the two calls.  dx is bitwise that of pdw_dwconv_dgrad; dw is the same sum
 * taken over other pieces of the images, so it can differ from pdw_dwconv_wgrad's in the last bit, and is the same from call to call. */
int pdw_dwconv_bwd(const void *gy, const void *w, const void *x, void *dx, void *dw, void *workspace, size_t workspace_bytes,
                   int B, int H, int W, int C, int KH, int KW, int SH, int SW, int PH, int PW, int DH, int DW, int dtype,
                   void *stream);

/* pdw_dwconv_wgrad for callers that cannot allocate device memory (code under HIP graph capture, tight serving
 * loops, harnesses that forbid hipMalloc): same arguments and bitwise the same result, but the fp32 partial sums
 * go to a buffer of pdw_static_scratch_bytes() (32 MiB) that is part of the library's device image instead of a
 * caller-supplied workspace.  The call allocates and frees nothing.  Extents whose
 * pdw_dwconv_wgrad_workspace_bytes exceeds that size are rejected with an error (use pdw_dwconv_wgrad).  Every
 * call on a device shares that device's one buffer, so calls that overlap on one device (two streams, two host
 * threads) race; the kernels overwrite what they read of it, nothing has to be cleared between calls.  Not
 * available between pdw_reduce_defer_begin and the flush.  The buffer's address on the current device is looked
 * up on the first call there (hipGetSymbolAddress); pdw_static_scratch_init() does that ahead of time, e.g.
 * before a graph capture begins.  No counterpart in the reference. */
size_t pdw_static_scratch_bytes(void);
int pdw_static_scratch_init(void);
int pdw_dwconv_wgrad_static(const void *x, const void *gy, void *dw, int B, int H, int W, int C, int KH, int KW,
                            int SH, int SW, int PH, int PW, int DH, int DW, int dtype, void *stream);

/* Two pdw_dwconv_wgrad calls of one pyramid block as one call: the same batch, channel count and odd square
 * filter (stride 1, padding K/2, dilation 1) on two tensors of different extents, each with its own workspace
 * (sized by pdw_dwconv_wgrad_workspace_bytes).  For 16-bit types the two problems share one launch, the second
 * one's workgroups starting as compute units finish with the first; otherwise this is the two calls in turn.
 * Results are bitwise those of the separate calls.  Replaces the two launches of
 * _depthwise_conv_weight_grad_kernel (dwconv_triton.py:377-385) that the backward of conv_block.py:41 makes
 * for the block's two scales. */
int pdw_dwconv_wgrad_pair(const void *x0, const void *gy0, void *dw0, void *workspace0, size_t workspace0_bytes,
                          int H0, int W0, const void *x1, const void *gy1, void *dw1, void *workspace1,
                          size_t workspace1_bytes, int H1, int W1, int B, int C, int K, int dtype, void *stream);
/* The three convolution launches at the end of a two-scale block's backward pass that do not depend on one another, as
 * one launch (backward of conv_block.py:14-16, 41 under autograd): dx = the full scale's input gradient from gy0 and w0
 * plus a quarter of gp per 2x2 block (what pdw_dwconv_dgrad_addpool computes; gp [B,H/2,W/2,C] is the pooled scale's
 * input gradient), dw0 = the full scale's weight gradient from x0 and gy0, dw1 = the half scale's from x1 and gy1
 * [B,H/2,W/2,C].  Square odd filter, stride 1, padding K/2, even H and W; workspaces as for the two pdw_dwconv_wgrad
 * calls.  Status 3 (nothing launched) when the fused kernel does not cover the case (fp32, C % 16, images narrower than
 * 33 columns...): the caller then makes the three calls.  dx is bitwise that of the separate call; the weight gradients
 * are the same sums taken over other pieces of the images (the launch cuts its three problems in its own way, into one
 * round of the chip where that is possible), so they can differ from pdw_dwconv_wgrad's in the last bit, and are
 * the same from call to call.  Between pdw_reduce_defer_begin/flush the two summations are recorded like any other. */
int pdw_dwconv_bwd3(const void *gy0, const void *w0, const void *gp, void *dx, const void *x0, void *dw0,
                    void *workspace0, size_t workspace0_bytes, const void *x1, const void *gy1, void *dw1,
                    void *workspace1, size_t workspace1_bytes, int B, int H, int W, int C, int K, int dtype,
                    void *stream);
/* Host only: the cut pdw_dwconv_bwd3 would choose for these extents (launch planning of the same call sites; no
 * reference counterpart, the Triton grid is fixed at dwconv_triton.py:318-333).  bands[0..2] receive the number of
 * pieces per image (rounded up: a piece may span images) of the input gradient, the full scale's and the half scale's
 * weight gradient (each >= 1).  Returns 0,
 * 3 when pdw_dwconv_bwd3 does not cover the case, 1 on invalid arguments.  Touches no device. */
int pdw_dwconv_bwd3_plan(int B, int H, int W, int C, int K, int dtype, int *bands);

/* The forward convolutions of both scales of a two-scale block as one launch (conv_block.py:14-16 at scales 1 and
 * 1/2): y0 = conv(x0, w0) on [B,H,W,C] and y1 = conv(x1, w1) on [B,H/2,W/2,C], x1 being an input (the caller's 2x2
 * average pool of x0, pdw_avgpool_fwd).  Square odd filter, stride 1, padding K/2, even H and W.  Status 3 (nothing
 * launched) when the fused kernel does not cover the case (fp32, C % 8, images narrower than 33 columns;
 * pdw_dwconv_fwd2_supported says so beforehand, so that a caller can have the full scale's convolution write the pool
 * instead: pdw_dwconv_fwd_pool): the caller then makes two pdw_dwconv_fwd calls.  Results are bitwise those of the
 * separate calls. */
int pdw_dwconv_fwd2_supported(int B, int H, int W, int C, int K, int dtype); /* 1: pdw_dwconv_fwd2 takes the case */
int pdw_dwconv_fwd2(const void *x0, const void *w0, void *y0, const void *x1, const void *w1, void *y1, int B, int H,
                    int W, int C, int K, int dtype, void *stream);
/* pdw_dwconv_fwd2 with the block's mean branch in B more workgroups of the same launch (conv_block.py:46-49:
 * m[b] = mean of x over the positions, rounded; rowbias[b] = m[b] w_pool^T + b_pool + b_out in fp32, the row that
 * pdw_dense_fwd adds to every output row of image b), from the sums of x over groups of positions that conv_up's
 * kernel left in parts [B][nparts][D] (pdw_dense_fwd_colsum): what pdw_pool_branch_fwd_parts computes, bitwise.  The
 * branch is three dependent trips to memory and a few kilobytes; in a launch of its own, or in one that saturates the
 * memory system, it costs microseconds, here it runs beside the convolutions.  Status 3 (nothing launched) where
 * pdw_dwconv_fwd2 does not take the case or the branch is not covered (D % 8, D > 128).  ldy0 = ldy1 = 0: the
 * convolution outputs y0, y1 as pdw_dwconv_fwd2 writes them; both > 0: the gated outputs of pdw_dwconv_fwd2_gate at these
 * pixel strides and channel offsets (inference). */
int pdw_dwconv_fwd2_mean(const void *x0, const void *w0, void *y0, int ldy0, int ych0, const void *x1, const void *w1,
                         void *y1, int ldy1, int ych1, int B, int H, int W, int C, int K, const float *parts,
                         int nparts, const void *w_pool, const void *b_pool, const void *b_out, void *m,
                         float *rowbias, int P, int D, int dtype, void *stream);

/* pdw_dwconv_fwd2 with the gate of pdw_dwconv_fwd_gate applied in the store of each scale (inference: neither
 * convolution output reaches HBM): y0[b,i,j, ych0 + c] and y1[b,i,j, ych1 + c], c < C/2, at pixel strides of ldy0 / ldy1
 * channels (0: C/2).  Covered where pdw_dwconv_fwd2 is and C % 16 == 0, strides and offsets multiples of 8;
 * status 3 otherwise (the caller then makes two pdw_dwconv_fwd_gate calls).  Results bitwise those calls'. */
int pdw_dwconv_fwd2_gate(const void *x0, const void *w0, void *y0, int ldy0, int ych0, const void *x1, const void *w1,
                         void *y1, int ldy1, int ych1, int B, int H, int W, int C, int K, int dtype, void *stream);

/* Adaptive average pooling x[B,H,W,C] -> y[B,h,w,C]; bin i covers [floor(i*H/h), ceil((i+1)*H/h)).
 * Replaces F.adaptive_avg_pool2d at conv_block.py:16 and the launch at avgpool_triton.py:225-229
 * (kernel :14-107; integer bin arithmetic here instead of the fp16 one at :42-47). */
int pdw_avgpool_fwd(const void *x, void *y, int B, int H, int W, int C, int h, int w, int dtype, void *stream);

/* Its gradient gy[B,h,w,C] -> gx[B,H,W,C], gather form (no atomics).  With accumulate != 0 the result
 * is added to gx (fp32 add, one rounding), otherwise gx is fully overwritten.
 * Replaces avgpool_triton.py:253-257 (kernel :118-203). */
int pdw_avgpool_bwd(const void *gy, void *gx, int B, int H, int W, int C, int h, int w, int accumulate, int dtype,
                    void *stream);

/* Bilinear resize, align_corners=False, no explicit scale factor: x[B,h,w,C] -> y[B,H,W,C].  Output pixels are
 * ldy elements apart (0 = dense, ldy = C), so the result can be written into a channel slice of a wider tensor
 * (the torch.cat of conv_block.py:43).
 * Replaces F.interpolate at conv_block.py:21 and the launch at up_triton.py:157-161 (kernel :14-125). */
int pdw_bilinear_fwd(const void *x, void *y, int B, int h, int w, int C, int H, int W, int ldy, int dtype,
                     void *stream);

/* Its gradient gy[B,H,W,C] (pixels ldgy elements apart, 0 = dense) -> gx[B,h,w,C], transpose of the above in
 * gather form.  The reference has no backward for up_triton.py; inside ConvBlock autograd supplies
 * upsample_bilinear2d_backward. */
int pdw_bilinear_bwd(const void *gy, void *gx, int B, int h, int w, int C, int H, int W, int ldgy, int dtype,
                     void *stream);

/* Gate  y[m,c] = x[m,c] * x[m,G+c] * sqrt(G),  G = I/2,  x[M,I] -> y[M,G] with rows ldy elements apart
 * (0 = dense)   (conv_block.py:10,18-19). */
int pdw_gate_fwd(const void *x, void *y, long long M, int I, int ldy, int dtype, void *stream);
/* gx[m,c] = gy*x[m,G+c]*sqrt(G);  gx[m,G+c] = gy*x[m,c]*sqrt(G); gy rows ldgy elements apart (0 = dense). */
int pdw_gate_bwd(const void *x, const void *gy, void *gx, long long M, int I, int ldgy, int dtype, void *stream);

/* Gate followed by the bilinear resize, in one pass: x[B,h,w,I] -> y[B,H,W,I/2], pixels of y ldy elements apart
 * (0 = dense).  Each gate value is rounded to the storage type before it is interpolated, as when pdw_gate_fwd
 * and pdw_bilinear_fwd run one after the other; the gated tensor itself is never written.
 * Replaces conv_block.py:18-21 for a branch with scale_factor != 1. */
int pdw_gate_bilinear_fwd(const void *x, void *y, int B, int h, int w, int I, int H, int W, int ldy, int dtype,
                          void *stream);
/* Gradient of the pair for exactly doubled extents (H = 2h, W = 2w, h,w >= 2; anything else is an error and the
 * caller runs pdw_bilinear_bwd then pdw_gate_bwd): gy[B,H,W,I/2] (pixels ldgy apart) and the gate's input
 * x[B,h,w,I] -> gx[B,h,w,I].  What autograd derives for conv_block.py:18-21. */
int pdw_bilinear_gate_bwd(const void *gy, const void *x, void *gx, int B, int h, int w, int I, int H, int W,
                          int ldgy, int dtype, void *stream);

/* The two gates of a block with scales (1, s) in one launch: y[..., 0:G] = gate(xf[B,H,W,I]) and
 * y[..., G:2G] = bilinear(gate(xh[B,h,w,I])) -> (H,W), G = I/2, pixels of y ldy elements apart (0 = 2G): the
 * torch.cat of conv_block.py:43 written directly (conv_block.py:18-21 for both entries of self.gates). */
int pdw_gate_pair_fwd(const void *xf, const void *xh, void *y, int B, int H, int W, int h, int w, int I, int ldy,
                      int dtype, void *stream);
/* Its gradient, one launch for any extents (exactly doubled ones take a kernel with fixed taps): gy[B,H,W,2G] (pixels
 * ldgy apart) -> gxf[B,H,W,I], gxh[B,h,w,I]; the same bits as pdw_gate_bwd on the first half and pdw_bilinear_bwd +
 * pdw_gate_bwd on the second. */
int pdw_gate_pair_bwd(const void *gy, const void *xf, const void *xh, void *gxf, void *gxh, int B, int H, int W,
                      int h, int w, int I, int ldgy, int dtype, void *stream);

/* Per-image sum over positions: x[B,P,C] -> out[B,C] (fp32), two deterministic passes through `workspace`.
 * Replaces x.mean(dim=(1,2)) at conv_block.py:46 (divide by P on the host side) and, in the backward, the
 * reduction of the broadcast add at conv_block.py:49. */
size_t pdw_spatial_sum_workspace_bytes(int B, int P, int C);
int pdw_spatial_sum(const void *x, float *out, void *workspace, size_t workspace_bytes, int B, int P, int C,
                    int dtype, void *stream);

/* In place y[b,p,c] += v[b,c] (v fp32 [B,C]): the broadcast add of the pooled branch, conv_block.py:49,
 * and its mirror in the backward (the gradient of the mean, conv_block.py:46). */
int pdw_add_rowbias(void *y, const float *v, int B, int P, int C, int dtype, void *stream);

/* Pooled branch of the block, forward (conv_block.py:46-47 plus the bias of :44): per image b,
 *   m[b,:]       = mean over the P positions of x[b,:,:]            (rounded to the element type, kept for backward)
 *   rowbias[b,o] = sum_c m[b,c] * w_pool[o,c] + b_pool[o] + b_out[o] (fp32; b_pool / b_out may be NULL)
 * rowbias is what pdw_dense_fwd / pdw_add_rowbias then broadcast over the positions (conv_block.py:49). */
size_t pdw_pool_branch_workspace_bytes(int B, int P, int D);
int pdw_pool_branch_fwd(const void *x, const void *w_pool, const void *b_pool, const void *b_out, void *m,
                        float *rowbias, void *workspace, size_t workspace_bytes, int B, int P, int D, int dtype,
                        void *stream);
/* Its backward from gy[B,P,D]: gbias[o] = sum over all positions of gy (the gradient of both biases; gbias2,
 * if not null, receives a second copy so that each bias owns its gradient tensor),
 * gw_pool[o,c] = sum_b gs[b,o] * m[b,c] with gs the per-image column sums of gy, and
 * dmean[b,c] = (1/P) * sum_o gs[b,o] * w_pool[o,c] (fp32), the per-image term that the mean's gradient
 * adds to every position of dx. */
int pdw_pool_branch_bwd(const void *gy, const void *m, const void *w_pool, void *gbias, void *gbias2, void *gw_pool,
                        float *dmean, void *workspace, size_t workspace_bytes, int B, int P, int D, int dtype,
                        void *stream);

/* The same two steps from per-chunk column sums the caller already has (parts[B][nparts][D], fp32, chunks of
 * equal or unequal length covering the P positions of an image), e.g. from pdw_dense_fwd_colsum: x / gy is not
 * read again.  pdw_pool_branch_bwd_parts still takes the workspace of pdw_pool_branch_workspace_bytes. */
int pdw_pool_branch_fwd_parts(const float *parts, int nparts, const void *w_pool, const void *b_pool,
                              const void *b_out, void *m, float *rowbias, int B, int P, int D, int dtype,
                              void *stream);
int pdw_pool_branch_bwd_parts(const float *parts, int nparts, const void *m, const void *w_pool, void *gbias,
                              void *gbias2, void *gw_pool, float *dmean, void *workspace, size_t workspace_bytes,
                              int B, int P, int D, int dtype, void *stream);

/* The middle of a two-scale block as one launch each way: pdw_gate_pair_fwd together with
 * pdw_pool_branch_fwd_parts, and pdw_gate_pair_bwd together with pdw_pool_branch_bwd_parts (same arguments, same
 * results; the mean branch is a handful of latency-bound workgroups that ride in the gate kernel's grid).  When
 * the combination is not covered (fp32, D > 128, unaligned slices) the two kernels are launched one after the
 * other.  P = positions per image of the tensor whose chunk sums `parts` holds (conv_block.py:40-49).  Between
 * pdw_reduce_defer_begin and the flush, pdw_block_mid_bwd leaves gw_pool, gbias and gbias2 to the deferred work
 * (they are sums over the images of values it writes into `workspace`, which must stay in place until then). */
int pdw_block_mid_fwd(const void *xf, const void *xh, void *y, int B, int H, int W, int h, int w, int I, int ldy,
                      const float *parts, int nparts, const void *w_pool, const void *b_pool, const void *b_out,
                      void *m, float *rowbias, int P, int D, int dtype, void *stream);
int pdw_block_mid_bwd(const void *gy, const void *xf, const void *xh, void *gxf, void *gxh, int B, int H, int W,
                      int h, int w, int I, int ldgy, const float *parts, int nparts, const void *m,
                      const void *w_pool, void *gbias, void *gbias2, void *gw_pool, float *dmean, void *workspace,
                      size_t workspace_bytes, int P, int D, int dtype, void *stream);
/* The middle of the two-scale block at inference: the gated half-resolution scale xh[B,h,w,G] upsampled
 * (pdw_bilinear_fwd) into y[..., :G] with pixel stride ldy (its slice of the concatenation), together with
 * pdw_pool_branch_fwd_parts, in one launch where the combination is covered and one after the other otherwise.
 * conv_block.py:20-21, :46-49. */
int pdw_block_mid_infer(const void *xh, void *y, int B, int H, int W, int h, int w, int G, int ldy,
                        const float *parts, int nparts, const void *w_pool, const void *b_pool, const void *b_out,
                        void *m, float *rowbias, int P, int D, int dtype, void *stream);

/* Dense layers of the block on the matrix cores.  bf16/fp16 with K <= 128, NO <= 128, K % 8 == 0, NO % 8 == 0 run the
 * tiled kernels (persistent workgroups, weights in LDS, a 32-row tile per wavefront over all features); wider ones
 * (K % 8 == 0, NO % 8 == 0) run tiles of 128 x 128 results, fp32 layers (K % 4 == 0, NO % 4 == 0) tiles of 64 x 64,
 * and fp32 weight gradients and other 16-bit widths (K % 4 == 0, NO % 4 == 0, K <= 256) one 32 x 32 result tile per
 * wavefront.  pdw_dense_supported says whether a shape is covered, forward, input gradient and weight gradient
 * alike - callers use a library GEMM otherwise; it answers no for fp32 with K > 256, which pdw_dense_fwd and
 * pdw_dense_wgrad take all the same.
 *   y[n,o] = sum_k x[n,k] * W(o,k) + bias[o] + rowbias[n / P][o]        x[N,K] -> y[N,NO]
 * W(o,k) = w[o*K + k] (w_kmajor == 0, the nn.Linear layout) or w[k*NO + o] (w_kmajor != 0, which gives the
 * input gradient of a layer from its own weight without a transpose).  bias (element type) and rowbias
 * (fp32 [ceil(N/P), NO]) may be NULL.  Replaces nn.Linear at conv_block.py:37 and :44 together with the
 * broadcast add of conv_block.py:49, and the matching input-gradient GEMMs of the backward. */
int pdw_dense_supported(int K, int NO, int dtype);
int pdw_dense_fwd(const void *x, const void *w, int w_kmajor, const void *bias, const float *rowbias, void *y,
                  long long N, int K, int NO, int P, int dtype, void *stream);

/* pdw_dense_fwd that also writes colsum[t][k] = sum of x[n,k] over the rows n of the t-th group of R rows (fp32,
 * ceil(N/R) x K, R = pdw_dense_colsum_rows(), the kernel's row tile): with R | P these are per-chunk sums of each
 * image, which pdw_pool_branch_fwd_parts /
 * _bwd_parts take in place of a second pass over x (the x.mean of conv_block.py:46 and its gradient ride on
 * conv_up, conv_block.py:37, and on the input gradient of conv_out, conv_block.py:44).  K = 64 or 128 only:
 * pdw_dense_colsum_supported. */
int pdw_dense_colsum_supported(int K, int NO, int dtype);
int pdw_dense_colsum_rows(void);
int pdw_dense_fwd_colsum(const void *x, const void *w, int w_kmajor, const void *bias, const float *rowbias, void *y,
                         float *colsum, long long N, int K, int NO, int P, int dtype, void *stream);

/* pdw_dense_fwd_colsum for the pixels of x[B,H,W,K] (no rowbias) that also writes the 2x2 average pool of y,
 * pool[B,H/2,W/2,NO] = what pdw_avgpool_fwd makes of y (conv_block.py:37 together with the pooling of conv_block.py:16
 * for the second scale: the convolutions of both scales can then start together, pdw_dwconv_fwd2).  The kernel's row
 * tiles are blocks of 4 image rows x 8 columns, so colsum[t] are the sums of x over such blocks (still H*W/32 per
 * image, image after image).  Status 3 (nothing launched) where not covered: 16-bit types, (K, NO) = (128, 64),
 * (96, 48) or (64, 32), H % 4 == 0, W % 8 == 0 only. */
int pdw_dense_fwd_colsum_pool(const void *x, const void *w, const void *bias, void *y, float *colsum, void *pool, int B,
                              int H, int W, int K, int NO, int dtype, void *stream);

/* The output layer of a two-scale block on rows made where they are multiplied (conv_block.py:18-21, 41-44 and :44
 * as one launch): y[b,i,j,:] = [ gate(cf[b,i,j]) | bilinear resize to H x W of gate(ch[b]) at (i,j) ] w^T + bias +
 * rowbias[b], with cf[B,H,W,I] and ch[B,H/2,W/2,I] the convolution outputs of the two scales, gate(v) = v[:I/2] *
 * v[I/2:] * sqrt(I/2) rounded to `dtype`, w[D][I], bias[D] or NULL, rowbias fp32 [B][D] or NULL.  cat[B,H,W,I] (or
 * NULL) receives the rows, which the backward pass reads again.  Bitwise what pdw_gate_pair_fwd (or pdw_block_mid_fwd)
 * followed by pdw_dense_fwd produce; the gated tensor is not read back from memory.  ldf > 0 (inference, after
 * pdw_dwconv_fwd2_gate): both scales arrive gated, cf[B,H,W,I/2] at a pixel stride of ldf values and ch[B,H/2,W/2,I/2],
 * only the resize is left to do and cat must be NULL.  Status 3 (nothing launched) where not covered
 * (pdw_dense_fwd_gated_supported says so beforehand): 16-bit types, H % 4 == 0, W % 8 == 0, I a multiple of 16 up to 64,
 * D a multiple of 8 up to 128 with D + 8 >= 1.5 I (I = 64, D = 128 runs the variant with compile-time extents). */
int pdw_dense_fwd_gated_supported(int H, int W, int I, int D, int dtype);
int pdw_dense_fwd_gated(const void *cf, const void *ch, void *cat, const void *w, const void *bias,
                        const float *rowbias, void *y, int B, int H, int W, int I, int D, int ldf, int dtype,
                        void *stream);

/* Weight gradient of such a layer: dw[m,o] = sum_n a[n,m] * b[n,o]  (a[N,M], b[N,NO] -> dw[M,NO]), fp32
 * accumulation, two deterministic passes through `workspace` (no atomics). */
size_t pdw_dense_wgrad_workspace_bytes(long long N, int M, int NO);
int pdw_dense_wgrad(const void *a, const void *b, void *dw, void *workspace, size_t workspace_bytes, long long N,
                    int M, int NO, int dtype, void *stream);

/* Both gradients of a dense layer y = x W^T (W[O][I]) that need gy, in one launch: dx[N,I] = gy W
 * (+ rowbias[n / P], fp32 [ceil(N/P), I], may be NULL; P >= 32) and dw[O,I] = gy^T x (workspace and summation as pdw_dense_wgrad, size pdw_dense_wgrad_workspace_bytes(N, O, I)); with
 * colsum != NULL also the sums of gy over groups of pdw_dense_colsum_rows() rows, as pdw_dense_fwd_colsum.  The two
 * products share the chip instead of following each other (each alone leaves half of it waiting on memory).
 * Covered (pdw_dense_bwd_pair_supported): 16-bit types and the widths pdw_dense_fwd and pdw_dense_wgrad both cover
 * (multiples of 8 up to 128, at most 8 tiles of 32 x 32 in dW); (O, I) = (128, 64), (64, 128), (64, 32), (32, 64) -
 * the backward of conv_out and conv_up, conv_block.py:44 and :37, in ConvBlock(128) and ConvBlock(64) - run with
 * the extents as compile-time constants; colsum where pdw_dense_bwd_pair_colsum_supported says so (the widths
 * pdw_dense_fwd_colsum covers); other shapes take pdw_dense_fwd(w_kmajor) and pdw_dense_wgrad.  Unlike pdw_dense_wgrad it carries no recorded summations along. */
int pdw_dense_bwd_pair_supported(int O, int I, int dtype);
int pdw_dense_bwd_pair_colsum_supported(int O, int I, int dtype); /* ... with the tile sums (`colsum` != NULL) */
int pdw_dense_bwd_pair(const void *gy, const void *w, const void *x, void *dx, float *colsum, void *dw, void *workspace,
                       size_t workspace_bytes, const float *rowbias, int P, long long N, int O, int I, int dtype,
                       void *stream);

/* The whole block of conv_block.py:25-49 (scales (1, 1/2), conv_up without bias) as one host call each way: the
 * launch sequence of the entry points above (forward: conv_up with the pool of its result, the convolutions of both
 * scales with the mean branch, conv_out on rows it makes from their outputs, writing cat: 3 launches for D = 128,
 * I = 64, H % 4 == 0, W % 8 == 0; other widths that pdw_dense_fwd_gated covers pool in a launch of their own; else the
 * gates and the mean branch are one launch before conv_out; backward: 5
 * launches and one summation launch)
 * without a host interpreter between them.  Covered when pdw_convblock_supported: 16-bit dtype, even H, W >= 4 with
 * H*W a multiple of pdw_dense_colsum_rows(), layer widths D (block), I (inner, a multiple of 16) that the dense
 * kernels and pdw_dense_bwd_pair cover (multiples of 8 up to 128; D = 128, 96 and 64 with I = D / 2 run variants with
 * compile-time extents), odd K.  All tensors channels-last and contiguous, all
 * parameters in `dtype`: x, y[B,H,W,D]; w_up[I,D]; w_dw0, w_dw1[K,K,I]; w_pool[D,D]; w_out[D,I]; b_pool, b_out[D] or
 * NULL.  The forward writes what the backward reads again: a = conv_up(x), c0 = conv(a), xp = pool(a)[B,H/2,W/2,I],
 * c1 = conv(xp), cat[B,H,W,I] (the gated scales), m[B,D] (per-image mean of x).  The backward overwrites dx and the
 * parameter gradients (gb_pool, gb_out may be NULL).  Workspaces: device scratch of the stated size, free for reuse
 * when the call's work on `stream` is done.  Results are bitwise those of the calls listed above made one by one.
 * Replaces the Python-level sequence of ConvBlock.forward, conv_block.py:36-49, and its autograd backward. */
int pdw_convblock_supported(int B, int H, int W, int D, int I, int K, int dtype);
/* Inference forward of the same block (same coverage): y only.  conv_up (which also pools its result for the second
 * scale where its kernel can, pdw_dense_fwd_colsum_pool); then, where pdw_dense_fwd_gated covers the widths and
 * extents, the convolutions of both scales with the mean branch in their launch (pdw_dwconv_fwd2_mean) and conv_out on
 * rows it makes itself from their outputs: three launches, no gated or concatenated tensor in memory.  Elsewhere, for
 * filters up to 13, each
 * scale's convolution with the gate applied in its store (both as one launch, pdw_dwconv_fwd2_gate, or
 * pdw_dwconv_fwd_gate twice, the full-resolution one then pooling its input), the half-resolution gate upsampled into
 * its slice of the concatenation with the mean branch (pdw_block_mid_infer), conv_out: neither convolution output is
 * written to HBM; larger filters at those widths run the launches of pdw_convblock_fwd on workspace tensors (measured
 * faster than the gated store of their 8-channel slices).  Every intermediate lives in `workspace`
 * (pdw_convblock_infer_workspace_bytes).  Same arithmetic as
 * pdw_convblock_fwd.  Replaces ConvBlock.forward under torch.no_grad(), conv_block.py:36-49 with :13-22. */
size_t pdw_convblock_infer_workspace_bytes(int B, int H, int W, int D, int I, int K, int dtype);
int pdw_convblock_infer(const void *x, const void *w_up, const void *w_dw0, const void *w_dw1, const void *w_pool,
                        const void *b_pool, const void *w_out, const void *b_out, void *y, void *workspace,
                        size_t workspace_bytes, int B, int H, int W, int D, int I, int K, int dtype, void *stream);
size_t pdw_convblock_fwd_workspace_bytes(int B, int H, int W, int D, int I, int K, int dtype);
int pdw_convblock_fwd(const void *x, const void *w_up, const void *w_dw0, const void *w_dw1, const void *w_pool,
                      const void *b_pool, const void *w_out, const void *b_out, void *a, void *c0, void *xp, void *c1,
                      void *cat, void *m, void *y, void *workspace, size_t workspace_bytes, int B, int H, int W,
                      int D, int I, int K, int dtype, void *stream);
size_t pdw_convblock_bwd_workspace_bytes(int B, int H, int W, int D, int I, int K, int dtype);
int pdw_convblock_bwd(const void *gy, const void *x, const void *a, const void *c0, const void *xp, const void *c1,
                      const void *cat, const void *m, const void *w_up, const void *w_dw0, const void *w_dw1,
                      const void *w_pool, const void *w_out, void *dx, void *gw_up, void *gw_dw0, void *gw_dw1,
                      void *gw_pool, void *gb_pool, void *gw_out, void *gb_out, void *workspace,
                      size_t workspace_bytes, int B, int H, int W, int D, int I, int K, int dtype, void *stream);

/* The two-scale block (scales 1 and s: pooled extents h, w; conv_up without bias) on every shape and type that the
 * library's dense and convolution kernels cover (fp32, odd extents, pooled sizes that are not exact halves, widths that
 * are not multiples of 16), as one host call each way; the fused launches of pdw_convblock_* where those cover the
 * shape.  Covered when pdw_block_supported.  `saved` is one device buffer of pdw_block_saved_bytes that the forward
 * fills and the backward reads (its layout is the library's own: everything between the two calls is in it); a forward
 * that no backward follows uses it as its workspace.  y is scratch of the forward until its last launch writes it, so it must
 * not overlap x.  x, y, gy, dx[B,H,W,D]; weights and their gradients as for
 * pdw_convblock_*; dx may be NULL (not wanted), gb_pool and gb_out too.  Status 3: case not covered, nothing launched.
 * Replaces ConvBlock.forward, conv_block.py:36-49, and its autograd backward. */
int pdw_block_supported(int B, int H, int W, int h, int w, int D, int I, int K, int dtype);
size_t pdw_block_saved_bytes(int B, int H, int W, int h, int w, int D, int I, int K, int dtype);
int pdw_block_fwd(const void *x, const void *w_up, const void *w_dw0, const void *w_dw1, const void *w_pool,
                  const void *b_pool, const void *w_out, const void *b_out, void *y, void *saved, size_t saved_bytes,
                  int B, int H, int W, int h, int w, int D, int I, int K, int dtype, void *stream);
size_t pdw_block_bwd_workspace_bytes(int B, int H, int W, int h, int w, int D, int I, int K, int dtype);
int pdw_block_bwd(const void *gy, const void *x, const void *saved, const void *w_up, const void *w_dw0,
                  const void *w_dw1, const void *w_pool, const void *w_out, void *dx, void *gw_up, void *gw_dw0,
                  void *gw_dw1, void *gw_pool, void *gb_pool, void *gw_out, void *gb_out, void *workspace,
                  size_t workspace_bytes, int B, int H, int W, int h, int w, int D, int I, int K, int dtype,
                  void *stream);

/* Norms over the channels of rows x[N][C], one row a pixel or token, and the gated residual that closes a block.  They go
 * before and after a mixing block (the reference's block has neither norm nor residual: conv_block.py:36-49 is what goes between).
 *
 *   PDW_NORM_LAYER   norm(v) = (v - mean v) / sqrt(mean (v - mean v)^2 + eps) * weight + bias
 *   PDW_NORM_RMS     norm(v) = v / sqrt(mean v^2 + eps) * weight + bias
 *   PDW_NORM_NONE    norm(v) = v * weight + bias
 *
 * 1 <= C <= PDW_NORM_MAX_CHANNELS; weight, bias and scale [C] or NULL (1, 0 and 1).  Statistics and sums are fp32, a result is
 * rounded once.  stats (optional, 2 N floats): each row's mean and reciprocal deviation, which the backward reads.  Tensors may
 * have any alignment.  All of it is one pass over the tensors, and one launch more for the sums over rows that are weights' gradients;
 * those are added in a fixed order (no atomics). */
enum { PDW_NORM_NONE = 0, PDW_NORM_RMS = 1, PDW_NORM_LAYER = 2 };
enum { PDW_ACT_NONE = 0, PDW_ACT_SIGMOID = 1, PDW_ACT_SILU = 2 };
#define PDW_NORM_MAX_CHANNELS 8192

/* y = norm(x); kind is not PDW_NORM_NONE. */
int pdw_norm_fwd(const void *x, const void *weight, const void *bias, void *y, float *stats, long long N, int C, int kind,
                 float eps, int dtype, void *stream);
/* gx, gweight, gbias from gy (each may be NULL: not wanted), x and what the forward left in stats.  Workspace: needed where
 * gweight or gbias is wanted. */
size_t pdw_norm_bwd_workspace_bytes(long long N, int C, int dtype);
int pdw_norm_bwd(const void *gy, const void *x, const void *weight, const float *stats, void *gx, void *gweight, void *gbias,
                 void *workspace, size_t workspace_bytes, long long N, int C, int kind, int dtype, void *stream);

/* out = x + scale * act(gate) * norm(y), and with next_kind other than PDW_NORM_NONE also next = norm'(out), the norm before
 * the block that follows (of out as it is before rounding).  gate: NULL; one row for P consecutive rows of x (an image's; N must be a
 * multiple of P); with P = 1, as without a gate, a value for each.  Gate rows are ldgate elements apart (0: C).  stats, next_stats: of y and of out. */
int pdw_residual_fwd(const void *x, const void *y, const void *gate, const void *scale, const void *weight, const void *bias,
                     const void *next_weight, const void *next_bias, void *out, void *next, float *stats, float *next_stats,
                     long long N, int C, long long P, long long ldgate, int act, int kind, int next_kind, float eps, int dtype,
                     void *stream);
/* The gradients, from those of out (gout) and, with a next norm, of next (gnext).  x is read only with a next norm.  gx [N][C] is written only with a next norm (without one it is gout itself); ggate like gate, dense.  Each result
 * may be NULL (not wanted).  Workspace: needed where any of ggate (with P > 1), gscale, gweight, gbias, gnext_weight, gnext_bias is
 * wanted. */
size_t pdw_residual_bwd_workspace_bytes(long long N, int C, long long P, int next_kind, int dtype);
int pdw_residual_bwd(const void *gout, const void *gnext, const void *x, const void *y, const void *gate, const void *scale,
                     const void *weight, const void *bias, const void *next_weight, const float *stats, const float *next_stats,
                     void *gx, void *gy, void *ggate, void *gscale, void *gweight, void *gbias, void *gnext_weight,
                     void *gnext_bias, void *workspace, size_t workspace_bytes, long long N, int C, long long P,
                     long long ldgate, int act, int kind, int next_kind, int dtype, void *stream);

/* The gated linear recurrence  h_t = a_t h_(t-1) + (1 - a_t) x_t,  a_t = sigmoid(g_t),  y_t = h_t,  along the second axis of
 * [O][T][W][I], each of the O * W * I chains by itself: the recursive counterpart of the depthwise convolution, whose reach is its
 * filter's (dwconv_triton.py:20-104).  An axis h of images [B][h][w][C] is O = B, T = h, W = w, I = C (dense tensors are faster as
 * W = 1, I = w * C), an axis w is O = B * h, T = w, W = 1.
 *
 * xs[3], gs[3] (host): the strides of x and g in elements, element (o, t, w, i) is x[o * xs[0] + t * xs[1] + w * xs[2] + i]; y and
 * gy are dense.  h0, last [O][W][I]: the state before the first and after the last step, fp32, either may be NULL (h0: 0).
 * lengths[O] (device, may be NULL): the chains of o have lengths[o] steps, clamped to 0..T; x, g and gy behind them are not read, and
 * y, gx and gg are 0 there.  reverse: from the last step to the first.  `states` (pdw_scan_states_bytes; NULL where no backward
 * follows): what the backward needs.  States and sums are fp32; y is rounded once.  A chain is composed in pieces, so a state
 * that overflows to infinity can come out as NaN further on.  Workspaces: pdw_scan_workspace_bytes (0: none needed). */
size_t pdw_scan_states_bytes(int O, long long T, int W, int I);
size_t pdw_scan_workspace_bytes(int O, long long T, int W, int I, int backward);
int pdw_scan_fwd(const void *x, const void *g, const float *h0, const int *lengths, void *y, float *last, float *states,
                 void *workspace, size_t workspace_bytes, int O, long long T, int W, int I, const long long *xs,
                 const long long *gs, int reverse, int dtype, void *stream);
/* gx, gg (at the strides gxs, ggs) and gh0 from gy and glast, either of which may be NULL (0), as may each result. */
int pdw_scan_bwd(const void *gy, const float *glast, const void *x, const void *g, const int *lengths, const float *states,
                 void *gx, void *gg, float *gh0, void *workspace, size_t workspace_bytes, int O, long long T, int W, int I,
                 const long long *xs, const long long *gs, const long long *gxs, const long long *ggs, int reverse, int dtype,
                 void *stream);
/* One step of B x C chains (a token for each of B streams): y = new_state = sigmoid(g) state + sigmoid(-g) x.  Rows of x and g are
 * ldx and ldg elements apart, the others dense.  new_state may be state itself, but must not overlap it otherwise. */
int pdw_scan_step(const void *x, const void *g, const float *state, float *new_state, void *y, long long B, int C,
                  long long ldx, long long ldg, int dtype, void *stream);

/* Norms of the rows of heads (queries, and keys where there are any) with the rotation by positions in the same pass.
 *   n = x (PDW_HEAD_NONE), x / sqrt(mean x^2 + eps) * weight (PDW_HEAD_RMS) or x / sqrt(sum x^2 + eps) * weight (PDW_HEAD_L2)
 * for each row of d channels (1 to PDW_HEAD_MAX_CHANNELS); the first 2 P channels of n, P the sum of the sections, are pairs, halves (i, P + i)
 * or (neighbours != 0) (2 i, 2 i + 1), and pair i is turned by position * frequency_i, the position along the axis in whose section i lies.
 * Tensor 0 has heads[0] heads, tensor 1 (may be NULL) heads[1]; element (token, head, i) of it is x[token * xt + head * xh + i].
 * Positions: NULL, tokens are a grid whose last axes have the extents grid[0..axes); or rows of `axes` numbers of position_type, one for each
 * of the last `positions_rows` tokens' places, repeated (token modulo rows).  Frequencies (device, fp32, radians, P of them): NULL, then
 * base^(-j / section) for pair j of each section.  Weights have the tensors' type; NULL: 1.  PDW_HEAD_NONE has none, and no gradients of any. */
enum { PDW_HEAD_NONE = 0, PDW_HEAD_RMS = 1, PDW_HEAD_L2 = 2 };
enum { PDW_POSITIONS_GRID = 0, PDW_POSITIONS_I32 = 1, PDW_POSITIONS_I64 = 2, PDW_POSITIONS_F32 = 3 };
#define PDW_HEAD_MAX_CHANNELS 256
typedef struct {
    const void *x[2], *weight[2];
    long long xt[2], xh[2];
    const void *positions;
    const float *frequencies;
    long long tokens, positions_rows;
    int heads[2], grid[3], sections[3], d, axes, kind, neighbours, position_type, dtype;
    float eps;
    double base;
} pdw_rotary;
/* y[0], y[1] dense [token][head][d]. */
int pdw_rotary_fwd(const pdw_rotary *call, void *const y[2], void *stream);
/* gx[2] (dense) and gweight[2] from gy[2] (dense); each result may be NULL.  Workspace: needed where a gweight is wanted (of no rows: zeros, without). */
size_t pdw_rotary_bwd_workspace_bytes(int d);
int pdw_rotary_bwd(const pdw_rotary *call, const void *const gy[2], void *const gx[2], void *const gweight[2], void *workspace,
                   size_t workspace_bytes, void *stream);

/* The gated delta rule along the second axis of [O][T][W][heads][..]: for each of the O * W * Hv chains a state S [dk][dv],
 *   u_t = beta_t (v_t - a_t S_(t-1)^T k_t),   S_t = a_t S_(t-1) + k_t u_t^T,   y_t = scale S_t^T q_t,
 * a = sigmoid(g), beta = sigmoid(b) (logits != 0) or a = exp(g), beta = b (g at most 0 by right).  q, k have Hk heads of dk channels, v and y Hv of dv,
 * g and b a number for each of Hv; value heads share key heads in groups of Hv / Hk.  dk, dv: 1 to PDW_DELTA_MAX_CHANNELS.
 * Element (o, t, w, head, i) is x[o * s[0] + t * s[1] + w * s[2] + head * s[3] + i].  y and the gradients are dense.
 * h0, last [O][W][Hv][dk][dv], fp32, either may be NULL; they must not overlap, nor may a backward's glast and gh0.  lengths[O] (device, may be NULL):
 * valid steps, limited to 0..T; what lies behind has no part in any result (of an empty sequence the first step is loaded
 * and dropped), y and the gradients are 0 there.  reverse: from the last valid step to the first.
 * gates_f32: g and b are fp32 whatever dtype is, and so are their gradients, which hold some 17 bits of the terms that they are sums of in 16-bit calls.
 * `states` (pdw_delta_states_bytes; NULL where no backward follows): what the backward needs.  States and sums are fp32; y is rounded once.  Products
 * are made of bf16 planes: infinities in k, q, v or a state come out as NaN (in calls that go step by step as a loop has them).  A value that is not
 * finite reaches what the rule hands it to, y of its own step and the later ones and the last state (in v: of its channel), and no other step, channel or
 * head; among the gradients it can reach all steps of its chunk of 64, and what the rule hands those to. */
#define PDW_DELTA_MAX_CHANNELS 128
typedef struct {
    const void *q, *k, *v, *g, *b;
    long long qs[4], ks[4], vs[4], gs[4], bs[4];
    const float *h0;
    const int *lengths;
    long long T;
    int O, W, Hk, Hv, dk, dv, reverse, logits, gates_f32, dtype;
    float scale;
} pdw_delta;
size_t pdw_delta_states_bytes(const pdw_delta *call);
size_t pdw_delta_workspace_bytes(const pdw_delta *call, int backward, int with_states);
int pdw_delta_fwd(const pdw_delta *call, void *y, float *last, void *states, void *workspace, size_t workspace_bytes, void *stream);
/* Gradients from gy (dense) and glast (may be NULL: 0); gh0 may be NULL, as may each of the others. */
int pdw_delta_bwd(const pdw_delta *call, const void *gy, const float *glast, const void *states, void *gq, void *gk, void *gv, void *gg,
                  void *gb, float *gh0, void *workspace, size_t workspace_bytes, void *stream);
/* The same step by step, for single tokens and a few: h0 is the state (NULL: 0), last the new one, which may be h0 itself, but must not overlap
 * it otherwise. */
int pdw_delta_step(const pdw_delta *call, void *y, float *last, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* PDW_H_ */
