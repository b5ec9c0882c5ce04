/*
 * n3d.h — C ABI of libn3d.so, the MI355X (gfx950) implementation of the Next3D generator-forward
 * hot path.  This is the drop-in boundary: every entry point replaces one native plugin function
 * or one ATen/third-party call of the reference (file:line cited per function; paths relative to
 * the reference root, `tat/` = training_avatar_texture/, `vr/` = tat/volumetric_rendering/).
 *
 * Conventions (mirroring the reference plugins):
 *   - plain pointers + sizes, no torch types; all pointers are DEVICE pointers unless noted;
 *   - inputs are borrowed, outputs are CALLER-allocated; the library never allocates, frees or
 *     synchronises; every kernel is enqueued on the `stream` argument (a hipStream_t);
 *   - return 0 on success, negative on error; n3d_last_error() gives the message (the Python
 *     wrapper raises RuntimeError, the analogue of TORCH_CHECK in bias_act.cpp:39-55);
 *   - tensors are float32, NCHW-contiguous unless a stride argument says otherwise.
 */
#ifndef N3D_H_
#define N3D_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef void* n3d_stream_t; /* hipStream_t */

#define N3D_ABI_VERSION 9

/* activation ids = the reference's cuda_idx (torch_utils/ops/bias_act.py:23-33) */
enum { N3D_ACT_LINEAR = 1, N3D_ACT_RELU = 2, N3D_ACT_LRELU = 3, N3D_ACT_TANH = 4, N3D_ACT_SIGMOID = 5,
       N3D_ACT_ELU = 6, N3D_ACT_SELU = 7, N3D_ACT_SOFTPLUS = 8, N3D_ACT_SWISH = 9 };
enum { N3D_F32 = 0, N3D_F16 = 1, N3D_BF16 = 2 /* the token operators only */ };
/* activation layouts: float32 NCHW; split8 (see n3d_fir4_split8); "c8" = float32 [N][C/8][H][row pitch in pixels][8], one
 * 32-byte unit = 8 consecutive channels of one pixel (what the transposed convolution hands to n3d_fir4_split8) */
enum { N3D_LAYOUT_NCHW_F32 = 0, N3D_LAYOUT_SPLIT8 = 1, N3D_LAYOUT_C8_F32 = 2,
       N3D_LAYOUT_H8_F16 = 3 /* "h8": float16 [N][C/8][H][W][8], dense — the activations of the reference's float16 blocks (n3d_conv2d_f16) */ };

int n3d_abi_version(void);
const char* n3d_last_error(void);

/* Per-kernel-family timing for bench.py's roofline leg.  While enabled, every entry point brackets its
 * kernel launches with HIP events recorded ON THE LAUNCH STREAM and books its algorithmic flops / bytes.
 * n3d_prof_read synchronises the recorded events and returns the totals for one family since the last reset. */
enum { N3D_K_BIAS_ACT = 0, N3D_K_UPFIRDN2D = 1, N3D_K_CONV2D = 2, N3D_K_FC = 3, N3D_K_RENDER = 4, N3D_K_RASTER = 5,
       N3D_K_MISC = 6, N3D_K_CONV2D_BF16X3 = 7 /* 3x3 split-bf16 kernels: MFMA-bound */,
       N3D_K_CONV1X1_BF16X3 = 8 /* 1x1 split-bf16 kernels (and the float16 toRGB): HBM-bound */,
       N3D_K_CONV2D_F16 = 9 /* 3x3 float16 kernels of the fp16 blocks (n3d_conv2d_f16): MFMA / HBM */,
       N3D_K_RENDER_RAYS = 10 /* n3d_render_rays(_ex): depth-bounds pre-pass + render_rays_kernel (texel gathers through L1 / L2 + the decoder) */, N3D_K_LAYER_NORM = 11, N3D_K_ROTARY = 12, N3D_K_ATTENTION = 13, N3D_K_COUNT = 14 };
int n3d_prof_enable(int on);
int n3d_prof_reset(void);
int n3d_prof_read(int family, double* total_ms, int64_t* launches, double* flops, double* bytes);

/* ---- bias_act: replaces bias_act_plugin.bias_act forward (torch_utils/ops/bias_act.cpp:36,
 *      kernel bias_act.cu:27-150).  y = clamp(act(x + b[(i/step_b) % size_b]) * gain).
 *      b may be NULL; clamp < 0 disables clamping; x and y may alias. */
int n3d_bias_act(const void* x, const void* b, void* y, int64_t numel, int size_b, int64_t step_b, int dtype,
                 int act, float alpha, float gain, float clamp, n3d_stream_t stream);

/* Fused per-element epilogue shared by upfirdn2d / conv2d (all optional, applied in this order):
 *   v = v * row_scale[n*O + o] * const_scale;  v += noise[oy*OW+ox] * (*noise_strength);  v += bias[o];
 *   v = act(v) * gain;  clamp;  [round to float16];  v += residual[n, o, oy, ox]                       */
typedef struct {
    const float* row_scale;       /* [N,O] (row pitch row_scale_stride; 0 = O) or NULL — demodulation coefficients,
                                     tat/networks_stylegan2.py:72-79                                              */
    const float* noise;           /* [OH,OW] or NULL (noise_const, :320-321)                                     */
    const float* noise_strength;  /* device scalar, required when noise != NULL                                  */
    const float* bias;            /* [O] or NULL                                                                 */
    const float* residual;        /* [N,O,OH,OW] (batch stride residual_batch_stride) or NULL                    */
    int64_t residual_batch_stride;
    int64_t row_scale_stride;     /* floats between consecutive samples of row_scale (0 = densely packed [N,O])   */
    float const_scale;            /* e.g. Conv2dLayer.weight_gain (tat/networks_stylegan2.py:174)                */
    int act;                      /* N3D_ACT_*                                                                   */
    float alpha, gain, clamp;     /* clamp < 0: none                                                             */
    const float* residual_up_filter; /* NULL, or 16 taps [4][4]: `residual` is then the LOW-resolution image
                                        [N,O,OH/2,OW/2] and is upsampled x2 on the fly exactly like
                                        upfirdn2d.upsample2d(residual, f) (up=2, padding (2,1,2,1), gain 4, no flip):
                                        the skip-image path img = upsample2d(img) + toRGB(x) of SynthesisBlock.forward
                                        (tat/networks_stylegan2.py:580-584) without materialising the upsampled image */
    int round_f16;                /* != 0: the value is rounded to float16 (nearest even) and widened again after the clamp, before
                                     the residual is added — the storage rounding of the reference's fp16 blocks
                                     (tat/networks_stylegan2.py:548-552: x.to(float16); every operator of such a block returns
                                     float16) on float32 arithmetic.  Supported by the pre-split kernels (split8 / c8 layouts),
                                     the 1x1 kernel and n3d_fir4_split8; other kernels reject it.  The float16-block kernels
                                     (n3d_conv2d_f16, n3d_fir4_h8) always store float16; for them the value 2 selects the rounding of
                                     the reference's OFF-GPU bias_act (_bias_act_ref on half tensors, torch_utils/ops/bias_act.py:93-122:
                                     x + b, leaky_relu, x * gain are separate float16 tensor ops) instead of bias_act.cu's single
                                     rounding — used to match the reference's own CPU run of its float16 branch. */
} n3d_epilogue;

/* ---- upfirdn2d: replaces upfirdn2d_plugin.upfirdn2d (torch_utils/ops/upfirdn2d.cpp:20, kernels
 *      upfirdn2d.cu:33,102).  x [N,C,H,W] -> y [N,C,OH,OW], f [fh,fw] float32 (2-D taps),
 *      OH = (H*upy + pady0 + pady1 - fh + downy) / downy (same for W).  `epi` may be NULL. */
int n3d_upfirdn2d(const float* x, const float* f, float* y, int N, int C, int H, int W, int fh, int fw, int upx,
                  int upy, int downx, int downy, int padx0, int padx1, int pady0, int pady1, int flip, float gain,
                  int64_t x_batch_stride, int64_t y_batch_stride, const n3d_epilogue* epi, n3d_stream_t stream);
/* Same, with explicit row pitches (floats; plane pitch = rows * pitch): x_row_stride >= W for the input, y_row_stride >= OW
 * (0 = OW) for the output.  Rows that start 16-byte aligned (pitch % 4 == 0) are fetched / stored with aligned 16-byte
 * accesses; a pitched output takes no per-pixel epilogue inputs (noise / residual).  The odd-width images of the model —
 * the (2W+1)-wide transposed-conv output in front of the up FIR, the (W+1)-wide FIR output in front of the stride-2 conv —
 * travel this way. */
int n3d_upfirdn2d_pitched(const float* x, const float* f, float* y, int N, int C, int H, int W, int64_t x_row_stride,
                          int64_t y_row_stride, int fh, int fw, int upx, int upy, int downx, int downy, int padx0, int padx1,
                          int pady0, int pady1, int flip, float gain, int64_t x_batch_stride, int64_t y_batch_stride,
                          const n3d_epilogue* epi, n3d_stream_t stream);

/* ---- filtered_lrelu: replaces filtered_lrelu_plugin.filtered_lrelu forward (torch_utils/ops/filtered_lrelu.cpp:20, kernel
 *      filtered_lrelu.cu:143-144; semantics of _filtered_lrelu_ref, filtered_lrelu.py:123-155) in ONE launch:
 *        y = upfirdn2d( clamp(lrelu(upfirdn2d(x + b[c], fu, up, pad, gain=up^2), slope) * gain), fd, down )
 *      x [N,C,H,W] -> y [N,C,OH,OW], OH = (H*up + py0 + py1 - (fuh-1) - (fdh-1) + (down-1)) / down (same for W).
 *      fu [fuh,fuw] / fd [fdh,fdw] float32 2-D taps, NULL = a single unit tap (sizes 1); b [C] or NULL; clamp < 0: none;
 *      flip as upfirdn2d's flip_filter.  The up-sampled intermediate stays in LDS. */
int n3d_filtered_lrelu(const float* x, const float* fu, const float* fd, const float* b, float* y, int N, int C, int H, int W,
                       int fuh, int fuw, int fdh, int fdw, int up, int down, int px0, int px1, int py0, int py1, float gain,
                       float slope, float clamp, int flip, n3d_stream_t stream);

/* ---- "split8": the activation layout of the pre-split convolution path.  A tensor [N,C,H,W] (C % 8 == 0) is stored as
 *        bf16  y[N][2 (hi, lo)][C/8][H][W][8]       hi = bf16(v), lo = bf16(v - float(hi))
 *      — 16-byte units of 8 consecutive channels of one pixel, the same 4 bytes per element as float32.  The PRODUCER of such a
 *      tensor does the operand split of the bf16x3 arithmetic (n3d_conv2d_bf16x3) and the consumer's style modulation once, in
 *      its epilogue; the consuming convolution then stages its operands with plain LDS-DMA copies.
 *      n3d_fir4_split8: the 4x4 FIR behind a transposed convolution (= n3d_upfirdn2d_pitched with up = down = 1, fh = fw = 4,
 *      padding 1, the layer epilogue `epi` fused: conv2d_resample.py:128-129 + bias_act) writing split8 instead of float32:
 *      x [N,C,H,W] float32 in the c8 layout (N3D_LAYOUT_C8_F32, row pitch x_row_stride pixels, 0 = W; batch stride in floats,
 *      0 = dense) -> y split8 [N,C,H-1,W-1], each value additionally multiplied by out_scale[n*out_scale_stride + c] (the
 *      next layer's style; NULL = 1). */
int n3d_fir4_split8(const float* x_c8, const float* f, void* y_split8, int N, int C, int H, int W, int64_t x_row_stride,
                    int64_t x_batch_stride, int flip, float gain, const n3d_epilogue* epi, const float* out_scale,
                    int64_t out_scale_stride, n3d_stream_t stream);
/* n3d_fir4_split8_sep: n3d_fir4_split8 for a separable filter f = outer(f1d, f1d) (f1d: 4 device floats; the caller's promise) and a
 * linear / leaky-ReLU epilogue: vertical pass, horizontal pass, 8 instead of 16 multiply-adds per output — the same float32 sum in
 * another order. */
int n3d_fir4_split8_sep(const float* x_c8, const float* f1d, void* y_split8, int N, int C, int H, int W, int64_t x_row_stride,
                        int64_t x_batch_stride, int flip, float gain, const n3d_epilogue* epi, const float* out_scale,
                        int64_t out_scale_stride, n3d_stream_t stream);
/* n3d_fir4_split8_nchw: the same kernel on a float32 NCHW input (row pitch x_row_stride floats, 0 = W; batch stride in floats, 0 =
 * dense) with `pad` (1 or 2) zero pixels on every side -> y split8 [N,C,H+2*pad-3,W+2*pad-3].  pad = 2 is the FIR in front of the
 * stride-2 convolution of Conv2dLayer(down=2) (upfirdn2d with padding [2,2,2,2], conv2d_resample.py:108-111): the down-sampling
 * layers then run on split8 input like the others. */
int n3d_fir4_split8_nchw(const float* x, const float* f, void* y_split8, int N, int C, int H, int W, int64_t x_row_stride,
                         int64_t x_batch_stride, int pad, int flip, float gain, const n3d_epilogue* epi, const float* out_scale,
                         int64_t out_scale_stride, n3d_stream_t stream);
/* n3d_fir4_split8_nchw_sep: n3d_fir4_split8_nchw for a separable filter f = outer(f1d, f1d) and a linear / leaky-ReLU epilogue (the
 * NCHW twin of n3d_fir4_split8_sep: column sums from the 8 channel planes, LDS, row pass). */
int n3d_fir4_split8_nchw_sep(const float* x, const float* f1d, void* y_split8, int N, int C, int H, int W, int64_t x_row_stride,
                             int64_t x_batch_stride, int pad, int flip, float gain, const n3d_epilogue* epi, const float* out_scale,
                             int64_t out_scale_stride, n3d_stream_t stream);
/* n3d_split8_from_nchw: a float32 NCHW tensor [N,C,HW] (dense planes, batch stride x_batch_stride floats, 0 = dense) ->
 * split8, every value multiplied by scale[n*scale_stride + c] first (the consumer's style; NULL = 1).  For tensors whose
 * producer cannot write split8 itself (two consumers that need different styles). */
int n3d_split8_from_nchw(const float* x, const float* scale, void* y_split8, int N, int C, int64_t HW, int64_t x_batch_stride,
                         int64_t scale_stride, n3d_stream_t stream);
/* 1 when n3d_conv2d_bf16x3 runs this 3x3 stride-1 float32-NCHW layer on the few-pixel kernel (conv2d_sk_bf16x3.hip: the whole K inside
 * one workgroup, one launch): ksplit / workspace are then ignored, the caller need not allocate one.  (N3D_CONV_SK=0: never.) */
int n3d_conv2d_sk_eligible(int N, int I, int O, int H, int W);
/* the same question for the few-pixel STRIDE-2 layers (ksize 3, mode 1, float32 NCHW in / out, dense rows, H x W = the INPUT image, odd): the <= 17 x 17
 * down-sampling layers of the mouth encoder (Conv2dLayer down = 2 behind its FIR, conv2d_resample.py:108-111) */
int n3d_conv2d_sk_s2_eligible(int N, int I, int O, int H, int W);
/* the same question for the few-position TRANSPOSED layers (ksize 3, mode 2, float32 NCHW in and out, one weight tensor for the batch): 1 = the one-launch
 * kernel takes the layer whatever `ksplit` says (no workspace needed) */
int n3d_conv2d_up_sk_eligible(int N, int I, int O, int H, int W);
/* Floats of `workspace` the few-pixel kernels (the three questions above; mode as n3d_conv2d_desc.mode, mode 1: H x W = the input image) use for this
 * layer when the descriptor carries arrival counters (desc.tickets), and the number of counters they need (*tickets_needed): 0 / 0 = not their layer,
 * or a layer whose grid covers the chip without slicing K. */
int64_t n3d_conv2d_sk_workspace(int N, int I, int O, int H, int W, int mode, int* tickets_needed);
/* 1 when n3d_conv2d_bf16x3 accepts a split8 input for this 3x3 stride-1 shape (x_layout = N3D_LAYOUT_SPLIT8), else 0.
 * n3d_conv2d_split8_ksplit: 0 = not accepted, 1 = accepted, > 1 = accepted and run with that split-K factor (layers whose pixel tiles
 * alone leave CUs idle: the caller then provides `workspace` = ksplit * N * O * H * W floats; desc.ksplit is ignored). */
int n3d_conv2d_split8_eligible(int N, int I, int O, int H, int W);
int n3d_conv2d_split8_ksplit(int N, int I, int O, int H, int W);

/* ---- conv2d weight preparation (done once per model): w [O,I,k,k] -> wt [k*k][I][OP] (K-major, the layout
 *      the MFMA kernel streams; OP = O rounded up to a multiple of 4, zero padded, so rows are 16-byte aligned)
 *      and, when wsq != NULL, wsq[o*I+i] = sum_k w[o,i,k]^2 (for demodulation). */
int n3d_conv2d_prep_weight(const float* w, float* wt, float* wsq, int O, int I, int ksize, n3d_stream_t stream);

/* ---- conv2d: the one dense contraction (fp32 MFMA implicit GEMM).  Replaces the ATen conv2d /
 *      conv_transpose2d calls issued by conv2d_resample (torch_utils/ops/conv2d_resample.py:96-136) inside
 *      modulated_conv2d (tat/networks_stylegan2.py:34-91) and Conv2dLayer (:173-183).
 *        mode 0: stride 1, padding ksize/2            y [N,O,H,W]
 *        mode 1: stride 2, padding 0 (ksize 3)        y [N,O,(H-3)/2+1,(W-3)/2+1]   (conv2d_resample.py:108-111)
 *        mode 2: transposed, stride 2 (ksize 3)       y [N,O,2H+1,2W+1]              (conv2d_resample.py:114-131)
 *      style [N,I] (or NULL) multiplies input channels (modulation); `epi` is the fused epilogue.
 *      ksplit > 1 splits the input channels over extra workgroups: partial sums go to `workspace`
 *      (ksplit*N*O*OH*OW floats) and a second kernel reduces + applies the epilogue. */
typedef struct {
    const float* x;      /* [N,I,H,W], batch stride x_batch_stride */
    const float* wt;     /* prepared weights [k*k][I][OP]          */
    const float* style;  /* [N,I] or NULL                          */
    float* y;            /* [N,O,OH,OW], batch stride y_batch_stride */
    float* workspace;    /* required when ksplit > 1               */
    int N, I, O, H, W;
    int ksize, mode, ksplit;
    int64_t x_batch_stride, y_batch_stride;
    int64_t style_stride; /* floats between consecutive samples of `style` (0 = densely packed [N,I]) */
    int64_t x_row_stride; /* floats between consecutive INPUT rows (0 = W).  Only the split-bf16 stride-2 kernel (mode 1) takes a
                             pitched input (the FIR output in front of it); every other kernel requires 0 / W */
    int64_t y_row_stride; /* floats between consecutive output rows (0 = OW).  A multiple of 4 >= OW gives the odd-width
                             (2W+1) transposed-conv output 16-byte-aligned rows for the FIR that follows */
    n3d_epilogue epi;
    int x_layout;         /* N3D_LAYOUT_NCHW_F32 (default) or, for n3d_conv2d_bf16x3 with ksize 3 / mode 0 or 2 (mode 2: c8 output only), N3D_LAYOUT_SPLIT8:
                             `x` then points to a split8 tensor that already carries the modulation (style must be NULL);
                             x_batch_stride still counts 4-byte elements (0 = dense) */
    int y_layout;         /* N3D_LAYOUT_NCHW_F32 (default) or, for the un-split transposed n3d_conv2d_bf16x3 (mode 2, O % 64 == 0,
                             demodulation-only epilogue), N3D_LAYOUT_C8_F32: y_row_stride then counts PIXELS (0 = OW) and
                             y_batch_stride floats (= O * OH * pitch); or, for the 1x1 n3d_conv2d_bf16x3 (O % 32 == 0),
                             N3D_LAYOUT_SPLIT8: y is the dense split8 tensor a following pre-split 3x3 layer reads (that layer's
                             style is NOT applied — plain Conv2dLayer consumers; y_batch_stride / y_row_stride ignored) */
    void* side_split8;    /* NULL, or (1x1 n3d_conv2d_bf16x3 with O <= 128, I % 32 == 0 — the toRGB layers) a second output: the INPUT x
                             multiplied by side_style [N,I] in the dense split8 layout, i.e. exactly n3d_split8_from_nchw(x, side_style):
                             a block's feature map has two readers (toRGB, and the next block's transposed convolution with ITS
                             styles, networks_stylegan2.py:469-475) and is read from HBM once for both.  With rgb_partial (below) on the 3x3
                             stride-1 kernel it is instead that layer's own OUTPUT times side_style [N,O] (O % 8 == 0) */
    const float* side_style;
    int64_t side_style_stride; /* floats between samples of side_style (0 = I) */
    int64_t wt_batch_stride;   /* BYTES between consecutive samples' prepared weights (a multiple of 16), 0 = one weight tensor shared by
                                  the batch.  Non-zero = PER-SAMPLE weights: what the FUSED branch of modulated_conv2d hands to F.conv2d /
                                  F.conv_transpose2d with groups = batch (tat/networks_stylegan2.py:82-88, conv2d_resample.py:96-136) —
                                  sample n of x is group n of the reference's [1, N*I, H, W] view, `wt` comes from
                                  n3d_conv2d_prep_weight_grouped.  Taken by n3d_conv2d (modes 0 / 2) and by n3d_conv2d_bf16x3's stride-1
                                  (NCHW or split8 input), transposed (NCHW) and 1x1 kernels; n3d_conv2d_f16's weights are per-sample by
                                  construction (this field is ignored there) */
    /* ---- ABI 6: toRGB fused into the LAST 3x3 layer of a network (SynthesisBlock.forward, tat/networks_stylegan2.py:575-584: the last block's
     *      x has ONE reader, its ToRGBLayer :353-357).  n3d_conv2d_bf16x3, ksize 3 / mode 0 / split8 input, no split-K: the kernel applies the
     *      layer epilogue to its tile and multiplies it, in float32, with rgb_weight [rgb_channels][O] (the toRGB layer's 1x1 weights) times
     *      rgb_style [N][O] (its styles, weight_gain included) — the partial colours of each 64-channel workgroup go to
     *      rgb_partial [N][ceil(O/64)][rgb_channels][H][W]; n3d_rgb_combine sums them and applies toRGB's own epilogue (bias, clamp, the skip image).
     *      y may then be NULL: the feature map itself (537 MB per step for the 512 x 512 layer at batch 4) is neither written nor read back.
     *      n3d_conv2d_f16 (mode 0) takes the same fields for a float16 block: rgb_weight = per-sample float16 toRGB weights [N][rgb_channels][O]
     *      (n3d_modulate_weights_f16, demodulate 0), rgb_style NULL; n3d_rgb_combine with epi.round_f16 applies n3d_torgb_h8's float16 epilogue. */
    const float* rgb_weight;   /* NULL (with rgb_partial NULL) = off */
    const float* rgb_style;
    float* rgb_partial;
    int rgb_channels;          /* 1 .. 4 */
    int64_t rgb_style_stride;  /* floats between samples of rgb_style (0 = O) */
    /* ---- ABI 7: arrival counters for kernels that split K over WORKGROUPS and reduce inside the launch (the few-pixel 3x3 layers of
     *      n3d_conv2d_bf16x3, conv2d_sk_bf16x3.hip): ticket_count zero-initialised 32-bit words owned by the caller, ONE pool per stream (launches of
     *      a stream are serialised; every launch leaves the words zero, so the pool is zeroed once at allocation).  With tickets != NULL and
     *      workspace = n3d_conv2d_sk_workspace(...) floats the layer's K is sliced over up to 256 workgroups and the last-arriving slice of an output
     *      tile adds the slices' slabs in slice order and applies the epilogue (bitwise reproducible); NULL = the whole K inside one workgroup. */
    unsigned int* tickets;
    int ticket_count;
} n3d_conv2d_desc;
int n3d_conv2d(const n3d_conv2d_desc* desc, n3d_stream_t stream);

/* ---- per-sample ("grouped") weight preparation for the operator boundary: ONE launch re-tiles the weights of all G groups of a
 *      grouped convolution into the layout a kernel family streams, group g at wt + g * (bytes per group):
 *        w : float32 (w_dtype N3D_F32) or float16 (N3D_F16) elements, element (g, o, i, tap) at w[g*stride_g + o*stride_o + i*stride_i + tap]
 *            — F.conv2d's [G*O, I, k, k] is (O*I*kk, I*kk, kk), F.conv_transpose2d's [G*I, O, k, k] is (I*O*kk, kk, O*kk);
 *        wt_kind 0: float32 K-major [G][k*k][I][OP] (n3d_conv2d; bytes per group = k*k*I*OP*4, OP = O rounded up to 4)
 *        wt_kind 1: split-bf16 tiles [G][k*k][I/16][2][2][OP64][8] (n3d_conv2d_bf16x3; k*k*I*OP64*4 bytes per group, I % 16 == 0)
 *        wt_kind 2: float16 tiles [G][9][I/16][2][O][8] (n3d_conv2d_f16; ksize 3, I % 16 == 0; 9*I*O*2 bytes per group) — a pure
 *                   re-tile for float16 input, one rounding for float32 input.
 *      Replaces nothing in the reference: ATen's grouped convolution reads [G*O, I, k, k] directly; here the matrix-core kernels
 *      stream K-major tiles, so the operator layer (torch_utils/ops/conv2d_gradfix.py) re-tiles once per call. */
int n3d_conv2d_prep_weight_grouped(const void* w, int w_dtype, void* wt, int wt_kind, int G, int O, int I, int ksize, int64_t stride_g,
                                   int64_t stride_o, int64_t stride_i, n3d_stream_t stream);

/* ---- conv2d, split-bf16 ("bf16x3") variant of mode 0 / ksize 3: every fp32 operand is split into hi + lo bf16 halves and
 *      a*b ~= a_hi*b_hi + a_hi*b_lo + a_lo*b_hi runs on v_mfma_f32_32x32x16_bf16 with fp32 accumulation (5.3x the fp32
 *      MFMA rate, ~2^-16 relative operand error; measured 8e-5 max-abs on the final RGB with every conv emulated this
 *      way).  Same descriptor as n3d_conv2d except `wt` = the split K-major weights from
 *      n3d_conv2d_prep_weight_bf16x3: bf16 [k*k][I/16][2 (hi,lo)][2 (k half)][OP64][8], OP64 = O rounded up to 64.
 *      Requires I % 16 == 0.  Same reference call sites as n3d_conv2d. */
int n3d_conv2d_prep_weight_bf16x3(const float* w, void* wt16, int O, int I, int ksize, n3d_stream_t stream);
int n3d_conv2d_bf16x3(const n3d_conv2d_desc* desc, n3d_stream_t stream);
/* y[n][c][h][w] = epilogue(sum_m partial[n][m][c][h][w]) — the second half of the fused toRGB above: `epi` is the toRGB layer's epilogue
 * (bias [C], clamp, residual = the skip image, with residual_up_filter the PREVIOUS block's half-resolution image, :580-584).  The M partial
 * images are added in index order: bitwise reproducible. */
int n3d_rgb_combine(const float* partial, float* y, int N, int M, int C, int H, int W, const n3d_epilogue* epi, n3d_stream_t stream);
/* Number of workgroups n3d_conv2d_bf16x3 launches for this shape at ksplit = 1 (its tile plan): the host picks a split-K
 * factor from it so that small layers still cover the 256 CUs. */
int n3d_conv2d_bf16x3_blocks(int N, int O, int H, int W, int mode);

/* ---- the reference's FLOAT16 blocks (super-resolution default route: `sr_num_fp16_res = 4` and no `force_fp32`,
 *      training/networks_stylegan2.py:417-452, tat/superresolution.py:264-290) on float16 matrix cores.  Activations travel in the
 *      "h8" layout (N3D_LAYOUT_H8_F16: float16 [N][C/8][H][W][8], C % 8 == 0, dense); every operator computes in float32 on float16
 *      inputs and rounds once on output, as the reference's half-precision CUDA ops do.
 *
 *      n3d_modulate_weights_f16: modulated_conv2d's FUSED branch (training/networks_stylegan2.py:53-66,88): per-sample weights
 *        w16[n] = half(weight * styles[n] (* dcoefs[n])) with the float16 pre-normalisation of :55-56 when demodulate != 0.
 *        w [O,I,k,k] float32, styles [N,I] (row pitch styles_stride floats, 0 = I).  Output: ksize 3 (I % 16 == 0) ->
 *        [N][9][I/16][2][O][8] float16 (the operand tiles n3d_conv2d_f16 streams); ksize 1 -> [N][O][I] (n3d_torgb_h8).
 *      n3d_conv2d_f16: F.conv2d / F.conv_transpose2d of that branch (conv2d_resample.py:96-136 with groups = N) — same descriptor
 *        as n3d_conv2d with x_layout = y_layout = N3D_LAYOUT_H8_F16, wt = n3d_modulate_weights_f16's output, style NULL, ksize 3,
 *        mode 0 (epilogue: [+noise] + bias, lrelu / linear, gain, clamp in the float16 order of SynthesisLayer.forward :320-329) or
 *        mode 2 (no epilogue: the float16 conv_transpose2d result, OH = 2H+1).  I % 16 == 0, O % 64 == 0, all strides 0 (dense).
 *      n3d_fir4_h8: upfirdn2d(x, f, padding 1, gain) behind the transposed convolution (conv2d_resample.py:128-129) + the layer's
 *        [noise] / bias_act (`epi`: bias, noise, act linear | lrelu, gain, clamp): h8 [N,C,H,W] -> h8 [N,C,H-1,W-1].  f [4,4] taps; f1d
 *        NULL, or 4 device floats with f == outer(f1d, f1d) (the caller's promise): the separable evaluation, same float32 sum.
 *      n3d_modulate_weights_f16_multi: up to 8 layers in one launch; `jobs` is a HOST array (copied into the kernel arguments),
 *        job j reads styles_base[n * styles_stride + styles_offset + i].
 *      n3d_torgb_h8: ToRGBLayer of a float16 block + `img = upsample2d(img) + y.to(float32)` (:446-451): x h8 [N,C,H,W], w16 [N][O][C]
 *        (n3d_modulate_weights_f16, ksize 1, demodulate 0, styles already times weight_gain), bias [O], img_lo [N,O,H/2,W/2] float32 or
 *        NULL, up_filter = the 4x4 taps (required with img_lo) -> img [N,O,H,W] float32.  C <= 512 (O <= 4: the image layers; larger O — the 32 / 96
 *        feature channels of the backbones' toRGB layers in float16 blocks — runs 16 output channels per workgroup); clamp < 0: none.
 *      n3d_cast_h8: float32 NCHW [N,C,HW] (batch stride x_batch_stride floats, 0 = dense) -> h8 (to_h8 != 0; `x.to(float16)` at the
 *        block entry, :437) or h8 -> dense float32 NCHW (to_h8 == 0). */
int n3d_modulate_weights_f16(const float* w, const float* styles, int64_t styles_stride, void* w16, int N, int O, int I, int ksize,
                             int demodulate, n3d_stream_t stream);
typedef struct {
    const float* w;          /* [O,I,k,k] float32 */
    void* w16;               /* output, layout as n3d_modulate_weights_f16 */
    int64_t styles_offset;   /* floats from styles_base to this layer's styles of sample 0 */
    int O, I, ksize, demodulate;
} n3d_modw_job;
int n3d_modulate_weights_f16_multi(const n3d_modw_job* jobs, int njobs, const float* styles_base, int64_t styles_stride, int N,
                                   n3d_stream_t stream);
int n3d_conv2d_f16(const n3d_conv2d_desc* desc, n3d_stream_t stream);
int n3d_fir4_h8(const void* x_h8, const float* f, const float* f1d, void* y_h8, int N, int C, int H, int W, int flip, float gain,
                const n3d_epilogue* epi, n3d_stream_t stream);
int n3d_torgb_h8(const void* x_h8, const void* w16, const float* bias, const float* img_lo, const float* up_filter, float* img, int N, int C,
                 int O, int H, int W, float clamp, n3d_stream_t stream);
int n3d_cast_h8(const void* x, void* y, int N, int C, int64_t HW, int64_t x_batch_stride, int to_h8, n3d_stream_t stream);
/* n3d_cast_h8_ex: the same with the NCHW side in float32 (nchw_dtype N3D_F32 = n3d_cast_h8) or float16 (N3D_F16: a pure layout change —
 * the operator boundary hands the float16 tensors of a reference fp16 block to n3d_conv2d_f16 and back this way). */
int n3d_cast_h8_ex(const void* x, void* y, int N, int C, int64_t HW, int64_t x_batch_stride, int to_h8, int nchw_dtype, n3d_stream_t stream);

/* ---- fully connected: replaces addmm / matmul+bias_act of FullyConnectedLayer.forward
 *      (tat/networks_stylegan2.py:114-127).  y[n,o] = post(act(sum_i pre(x[n,i]) * w[o,i] * wgain + b[o]*bgain)).
 *      pre_square: use x^2 (demodulation: sum_i s^2 * wsq);  post_rsqrt: y = rsqrt(y + 1e-8). */
int n3d_fc(const float* x, const float* w, const float* b, float* y, int N, int I, int O, float wgain, float bgain,
           int act, float alpha, float gain, int pre_square, int post_rsqrt, n3d_stream_t stream);

/* ---- batched fully connected: every style affine (and every demodulation coefficient) of one network in ONE launch.
 *      jobs: DEVICE array of n3d_fc_job; rows: DEVICE int32[total_rows][2] = (job index, output row within the job).
 *      For job j and sample n:  y_base[y_off + n*y_stride + o] = post(act(sum_i pre(x_base[x_off + n*x_stride + i]) *
 *      w[o*I + i] * wgain + b[o]*bgain)).  Same reference code as n3d_fc. */
typedef struct {
    const float* w;       /* [O,I] */
    const float* b;       /* [O] or NULL */
    int64_t x_off, x_stride, y_off, y_stride;
    int I, O;
    float wgain, bgain;
    int act;              /* N3D_ACT_* */
    float alpha, gain;
    int pre_square, post_rsqrt;
} n3d_fc_job;
int n3d_fc_multi(const n3d_fc_job* jobs, const int* rows, int total_rows, const float* x_base, float* y_base, int N,
                 n3d_stream_t stream);

/* ---- small element-wise pieces of the path.
 *      n3d_normalize_2nd_moment: y[r,:] = x[r,:] * rsqrt(mean(x[r,:]^2) + eps)  (tat/networks_stylegan2.py:27-29); y rows
 *        have pitch y_stride so two calls can fill the halves of the mapping network's concatenated input (:239-246).
 *        n3d_normalize_2nd_moment_f64: the same for a float64 x — the scripts' z is float64 (gen_samples_next3d.py:165) and MappingNetwork.forward
 *        converts it first (`z.to(torch.float32)`, :239): every element is rounded to float32, then the float32 arithmetic (bit-identical).
 *      n3d_truncate_ws: broadcast w [N,D] to ws [N,num_ws,D] and lerp the first `cutoff` latents towards w_avg with
 *        psi (MappingNetwork.forward :255-267; w_avg NULL or psi == 1 => plain broadcast).
 *      n3d_fma: y = a*b + c over a [NC,P] with b, c addressed as [nc*stride_nc + p*stride_p] (0 strides broadcast)
 *        (torch_utils/ops/fma.py:17-28 — only the non-fused modulated-conv branch uses it).
 *      n3d_to_uint8: (x*127.5+128).clamp(0,255) -> uint8 (gen_samples_next3d.py:201), layout preserved.
 *      n3d_layout_grid_u8: the video scripts' `layout_grid` helper in one pass (gen_videos_next3d.py:35-49, reenact_avatar_next3d.py:56-70:
 *        uint8 conversion, tiling and CHW -> HWC): frames [B,C,H,W] float32 (W % 4 == 0, B == cols * rows) -> uint8 canvas
 *        [rows*H, cols*W, C] (hwc = 1) or [C, rows*H, cols*W] (hwc = 0), frame b at tile row b / cols, tile column b % cols. */
int n3d_normalize_2nd_moment(const float* x, float* y, int rows, int D, int64_t y_stride, float eps, n3d_stream_t stream);
int n3d_normalize_2nd_moment_f64(const double* x, float* y, int rows, int D, int64_t y_stride, float eps, n3d_stream_t stream);
int n3d_truncate_ws(const float* w, const float* w_avg, float* ws, int N, int num_ws, int D, int cutoff, float psi,
                    n3d_stream_t stream);
int n3d_fma(const float* a, const float* b, const float* c, float* y, int64_t NC, int64_t P, int64_t b_nc, int64_t b_p,
            int64_t c_nc, int64_t c_p, n3d_stream_t stream);
int n3d_to_uint8(const float* x, unsigned char* y, int64_t numel, n3d_stream_t stream);
/* n3d_unpack_inputs: synthesis' input hand-over in one launch (tat/triplane_next3d.py:119-133: `v[:, :5023]`, `v[:, 5023:]`, `c[:, :16]`, `c[:, 16:25]`):
 * v [N][V + L][3] with batch stride v_batch_stride floats -> verts [N][V][3], lms [N][L][3]; c [N][>=25] with batch stride c_batch_stride ->
 * cam2world [N][16], intrinsics [N][9] — the dense tensors n3d_rasterize_views / n3d_render_rays_ex read. */
int n3d_unpack_inputs(const float* v, int64_t v_batch_stride, const float* c, int64_t c_batch_stride, float* verts, float* lms, float* cam2world,
                      float* intrinsics, int N, int V, int L, n3d_stream_t stream);
int n3d_layout_grid_u8(const float* frames, unsigned char* canvas, int B, int C, int H, int W, int cols, int rows, int hwc,
                       n3d_stream_t stream);
/* n3d_cast: float16 <-> float32 (N3D_F16 / N3D_F32), round to nearest even — the `x.to(dtype)` conversions at the
 * boundaries of the reference's fp16 blocks (tat/networks_stylegan2.py:548-552; tat/superresolution.py:210-217).  The
 * operator layer uses it to run fp16 tensors through the fp32-accumulating kernels: fp16 storage between operators,
 * exactly the rounding points of the reference's fp16 path. */
int n3d_cast(const void* x, void* y, int64_t numel, int src_dtype, int dst_dtype, n3d_stream_t stream);

/* ---- tri-plane blend (tat/triplane_next3d.py:171-174): planes = dyn * alpha + static * (1 - alpha), written
 *      CHANNELS-LAST [N,3,H,W,32] (one texel's 32 channels contiguous) for the renderer's gathers.
 *      front/side/top [N,32,H,W], stat [N,96,H,W], alpha [N,3,H,W]. */
int n3d_blend_planes(const float* front, const float* side, const float* top, const float* stat, const float* alpha,
                     float* planes_cl, int N, int H, int W, n3d_stream_t stream);
/* ... with alpha as the rasteriser leaves it: alpha_views [N,views,H,W] (n3d_rasterize_views' alpha4), plane p blended with the alpha image of view
 * v_p (front, side, top = views 0, 1, 3 of tat/triplane_next3d.py:140-145,226) — no index_select copy in between. */
int n3d_blend_planes_views(const float* front, const float* side, const float* top, const float* stat, const float* alpha_views,
                           float* planes_cl, int N, int H, int W, int views, int v_front, int v_side, int v_top, n3d_stream_t stream);
/* NCHW planes [N,3,32,H,W] -> channels-last, for callers holding blended planes in the reference layout. */
int n3d_planes_to_channels_last(const float* planes, float* planes_cl, int N, int H, int W, n3d_stream_t stream);

/* ---- volume renderer: replaces RaySampler.forward (vr/ray_sampler.py:24-63) + ImportanceRenderer.forward
 *      (vr/renderer.py:95-147: sample_stratified, sample_from_planes/grid_sampler_2d, OSGDecoder
 *      tat/triplane_next3d.py:359-371, MipRayMarcher2 vr/ray_marcher.py:27-66, sample_importance, sample_pdf,
 *      unify_samples).  One wavefront per ray; only feat [N,32,R,R] and depth [N,1,R,R] are written.
 *      tlin [Sc] = linspace(ray_start, ray_end, Sc); jitter [N,R*R,Sc] and u [N*R*R,Sf] are the uniform
 *      randoms the reference draws with torch.rand_like / torch.rand (vr/renderer.py:205,252);
 *      w1 [64,32] and w2t [64,34] are the decoder weights ALREADY multiplied by their weight_gain; w2t is the second
 *      layer TRANSPOSED (hidden-unit major) with each row padded by one zero (so a unit's 33 outgoing weights are
 *      contiguous, 8-byte aligned pairs);
 *      bounds_ws: 2 floats of scratch; wsum [N,R*R] optional (weights.sum(2)). */
int n3d_render_rays(const float* planes_cl, const float* cam2world, const float* intrinsics, const float* tlin,
                    const float* jitter, const float* u, const float* w1, const float* b1, const float* w2,
                    const float* b2, float* feat, float* depth, float* wsum, float* bounds_ws, int N, int R, int Sc,
                    int Sf, int PH, int PW, float depth_delta, float coord_scale, n3d_stream_t stream);
/* n3d_render_rays_ex: the renderer with the rendering options that lie outside the ffhq configuration (`opts` NULL = n3d_render_rays):
 *   white_back                 composite_rgb + 1 - weight_total (vr/ray_marcher.py:56-57);
 *   density_noise (+ draws)    sigma += randn * density_noise on every decoded sample (vr/renderer.py:152-153); the normal draws are INPUTS
 *                              like jitter / u: density_noise_coarse [N,R*R,Sc], density_noise_fine [N,R*R,Sf];
 *   disparity_space_sampling   coarse depths 1 / (1/ray_start * (1 - d) + 1/ray_end * d), d = linspace(0, 1, Sc) + jitter / (Sc - 1)
 *                              (vr/renderer.py:186-193): pass tlin = linspace(0, 1, Sc) and depth_delta = 1 / (Sc - 1);
 *   auto_bounds                ray_start = ray_end = 'auto' (vr/renderer.py:99-106): per-ray box entry / exit (math_utils.get_ray_limits_box
 *                              with box_side = rendering_kwargs['box_warp']), rays that miss the box repaired as the reference does, coarse
 *                              depths start + (end - start) * i / (Sc - 1) + jitter * (end - start) / (Sc - 1); tlin / depth_delta are
 *                              ignored; ray_bounds_ws = [N*R*R*2] floats of scratch (it holds every ray's (start, end) afterwards). */
typedef struct {
    int white_back;
    int disparity_space_sampling;
    float ray_start, ray_end;          /* disparity_space_sampling */
    int auto_bounds;
    float box_side;
    float* ray_bounds_ws;
    float density_noise;
    const float* density_noise_coarse;
    const float* density_noise_fine;
    /* ABI 7 — the seam between the two passes, for verification: the importance depths (sample_importance, vr/renderer.py:209-268) are
     * DISCONTINUOUS in the coarse pass's weights (a u that falls next to a CDF step lands in another bin for a last-bit difference), so an
     * end-to-end comparison of two correct implementations differs on a few rays.  fine_depths_out [N,R*R,Sf]: the depths this call sampled;
     * fine_depths_in [N,R*R,Sf]: use THESE instead of sampling (a checker feeds its own: everything behind the seam — second decode, merge,
     * march, composite — is then compared on identical samples, every ray).  Both NULL in normal use. */
    float* fine_depths_out;
    const float* fine_depths_in;
    /* ABI 8 — the decoder (OSGDecoder, tat/triplane_next3d.py:359-371) in the convolutions' split-bf16 arithmetic (three v_mfma_f32_32x32x16_bf16 per MAC, operand
     * truncation 2^-17) instead of float32-input MFMAs (bitwise an fmaf chain): 24 MFMAs of 8 passes per 32 samples instead of 67 of 16.  0 (and opts NULL): float32. */
    int decoder_split_bf16;
} n3d_render_opts;
int n3d_render_rays_ex(const float* planes_cl, const float* cam2world, const float* intrinsics, const float* tlin,
                       const float* jitter, const float* u, const float* w1, const float* b1, const float* w2,
                       const float* b2, float* feat, float* depth, float* wsum, float* bounds_ws, int N, int R, int Sc,
                       int Sf, int PH, int PW, float depth_delta, float coord_scale, const n3d_render_opts* opts, n3d_stream_t stream);

/* ---- point queries (shape extraction): replaces ImportanceRenderer.run_model (vr/renderer.py:149-155: sample_from_planes +
 *      OSGDecoder) as called by TriPlaneGenerator.sample / sample_mixed (tat/triplane_next3d.py:232-322).
 *      coords [N,M,3] world coordinates -> rgb [N,M,32], sigma [N,M,1]; coord_scale = 2 / box_warp; decoder weights as in
 *      n3d_render_rays (w1 [64,32], w2t [64,34], pre-scaled).  The reference's view directions are unused by the decoder. */
int n3d_sample_points(const float* planes_cl, const float* coords, const float* w1, const float* b1, const float* w2t,
                      const float* b2, float* rgb, float* sigma, int N, int64_t M, int PH, int PW, float coord_scale,
                      n3d_stream_t stream);

/* ---- mesh rasterisation of `views` orthographic views per sample: replaces TriPlaneGenerator.rasterize's
 *      geometry half (tat/triplane_next3d.py:193-216), Pytorch3dRasterizer.forward (vr/renderer.py:401-440, third-party
 *      pytorch3d rasterize_meshes) and fill_mouth (vr/renderer.py:583-602, third-party cv2.floodFill).
 *      verts [N,V,3], lms [N,Lm,3], rot [views,3,3] (angle2matrix), faces [F,3] int32 and face_uv [F,3,3] both with
 *      the reference's [0,2,1] vertex swap applied, uv_mask [mask_h,mask_w].
 *      Scratch: tv_ws [N*views*V*3] floats, zbuf_ws [N*views*H*W] uint64.
 *      Out: grid [N*views,H,W,2] (u,v), alpha [N*views,H,W] (mask*vis, hole-filled when fill != 0, view
 *      `binarize_view` additionally reduced to {0,1} as the reference's alpha_side), lm2d [N,Lm,2] (front view). */
int n3d_rasterize_views(const float* verts, const float* lms, const float* rot, const int* faces, const float* face_uv,
                        const float* uv_mask, int mask_h, int mask_w, float* tv_ws, unsigned long long* zbuf_ws,
                        float* grid, float* alpha, float* lm2d, int N, int V, int Lm, int F, int views, int H, int W,
                        float shift_x, float shift_y, float shift_z, float scale, int fill, int binarize_view,
                        n3d_stream_t stream);
/* ---- the two third-party calls of the rasterisation step under their own names, for reference code that runs UNRELOADED (boundary
 *      B1: a pickled model executes the reference's Pytorch3dRasterizer.forward / fill_mouth and imports pytorch3d / cv2 from
 *      next3d_amd/shims/):
 *      n3d_rasterize_meshes = pytorch3d.renderer.mesh.rasterize_meshes(meshes, image_size, blur_radius = 0, faces_per_pixel = 1,
 *        perspective_correct = False, cull_backfaces) as called at vr/renderer.py:415-424: verts_ndc [N,V,3] in PyTorch3D NDC, faces
 *        int32 [F,3] shared (faces_batch_stride 0) or [N,F,3] (stride 3F); zbuf_ws [N*H*W] uint64 scratch ->
 *        pix_to_face [N,H,W] int64 (packed n*F+f, -1 empty), zbuf [N,H,W] (-1 empty), bary [N,H,W,3] (-1 empty).  Same face kernel as
 *        n3d_rasterize_views.
 *      n3d_flood_fill = cv2.floodFill(img, mask, (0,0), new_val, lo_diff, up_diff, FLOODFILL_FIXED_RANGE) (vr/renderer.py:593) on N
 *        float32 images [N,H,W] (H, W <= 256), in place. */
int n3d_rasterize_meshes(const float* verts_ndc, const int* faces, int64_t faces_batch_stride, unsigned long long* zbuf_ws, long long* pix_to_face,
                         float* zbuf, float* bary, int N, int V, int F, int H, int W, int cull_backfaces, n3d_stream_t stream);
int n3d_flood_fill(float* images, int N, int H, int W, float new_val, float lo_diff, float up_diff, n3d_stream_t stream);
/* out [N,C,H,W] = grid_sample(textures [N,C,TH,TW], grid[:, view_a]) (+ the same for view_b when view_b >= 0)
 * — bilinear, zeros, align_corners=False, un-masked as in the reference (tat/triplane_next3d.py:218,225). */
int n3d_texture_project(const float* textures, const float* grid, float* out, int N, int C, int TH, int TW, int H, int W,
                        int views, int view_a, int view_b, n3d_stream_t stream);
/* The same for up to 4 planes in ONE launch: plane k = views view_a[k] (+ view_b[k] unless < 0) -> outs[k] [N,C,H,W].
 * (host arrays; the front / side / top planes of triplane_next3d.py:223-230 are one call) */
int n3d_texture_project_planes(const float* textures, const float* grid, float* const* outs, const int* view_a, const int* view_b,
                               int planes, int N, int C, int TH, int TW, int H, int W, int views, n3d_stream_t stream);
/* gen_mouth_mask (tat/triplane_next3d.py:330-344) on the device: lm2d [N,Lm,2] -> bbox [N,4] int32 (y0,y1,x0,x1). */
int n3d_mouth_bbox(const float* lm2d, int* bbox, int N, int Lm, n3d_stream_t stream);
/* F.interpolate(mode='bilinear', antialias=True, align_corners=False) = ATen _upsample_bilinear2d_aa
 * (tat/triplane_next3d.py:152,161; tat/superresolution.py:282-286) with optional per-sample DEVICE boxes
 * (y0,y1,x0,x1): src_box crops the source, dst_box restricts the written region (dst_square: region is s x s with
 * s = y1-y0, as the reference's paste at :161).  NULL box = whole tensor. */
int n3d_resize_aa(const float* src, float* dst, const int* src_box, const int* dst_box, int N, int C, int SH, int SW,
                  int DH, int DW, int dst_square, n3d_stream_t stream);
/* ... with an explicit batch stride of `src` in floats (0 = dense): a channel-slice view — the first 3 of the renderer's 32 feature channels as the RGB input of the
 * super-resolution module, tat/triplane_next3d.py:179-181 — is resized without a copy. */
int n3d_resize_aa_strided(const float* src, int64_t src_batch_stride, float* dst, const int* src_box, const int* dst_box, int N, int C, int SH, int SW,
                          int DH, int DW, int dst_square, n3d_stream_t stream);

/* ---- token operators: layer norm, rotary positions and attention over rows of channels (w vectors, tri-plane texels, frames of a video).  They have
 *      no counterpart in the reference.  dtype: N3D_F32 / N3D_F16 / N3D_BF16 as stated; element strides; every scratch buffer is the caller's. */

/* y = (x - mean) / sqrt(var + eps) * w + b over the last dimension: x [rows, C] with row stride x_stride (elements; channels dense) -> y [rows, C] dense.
 * w / b [C] or NULL, of w_dtype (N3D_F32 or dtype).  mean / rstd [rows] float32 for the gradient, both or neither NULL.  float32 statistics. */
int n3d_layer_norm(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, int64_t rows, int C, int64_t x_stride, int dtype,
                   int w_dtype, float eps, n3d_stream_t stream);
/* Gradients of n3d_layer_norm: dx [rows, C] dense (type dtype), dw / db [C] (type w_dtype); each may be NULL.  rows > 0.
 * workspace: n3d_layer_norm_bwd_workspace(rows, C, dtype) floats, needed when dw or db is asked for.  Sums in a fixed order: bitwise reproducible. */
int64_t n3d_layer_norm_bwd_workspace(int64_t rows, int C, int dtype);
int n3d_layer_norm_bwd(const void* dy, const void* x, const void* w, const float* mean, const float* rstd, void* dx, void* dw, void* db, float* workspace,
                       int64_t rows, int C, int64_t x_stride, int64_t dy_stride, int dtype, int w_dtype, n3d_stream_t stream);

/* Rotary positions with 1..4 axes.  Pairs of channels turn by position * base^-e: axis a owns sections[a] / 2 pairs, in order; the remaining
 * D - sum(sections) channels pass through.  e = 2 i / sections[a] for pair i of axis a, or (shared_ladder) p / P for pair p of all P.  A pair is
 * (2p, 2p + 1) when interleaved, else channels i and i + half — the halves of the axis's section, or of all rotated channels with shared_ladder.
 * inverse: turn back (the gradient).  q [B, L, heads_q, D] and k [B, L, heads_k, D] (heads_k 0: none) of one dtype with element strides (batch, token,
 * head) and dense channels -> out_q / out_k, dense.  positions: pos_type 0 float32, 1 int32, 2 int64; element (b, l, a) at
 * b * pos_batch_stride + l * pos_token_stride + a.  Angles in 64 bits. */
typedef struct {
    const void *q, *k, *positions;
    void *out_q, *out_k;
    int64_t q_strides[3], k_strides[3];
    int64_t pos_batch_stride, pos_token_stride;
    double base;
    int B, L, heads_q, heads_k, D, axes, sections[4];
    int dtype, pos_type, interleaved, shared_ladder, inverse;
} n3d_rotary_desc;
int n3d_rotary(const n3d_rotary_desc* desc, n3d_stream_t stream);

/* Attention.  q [B, Lq, heads_q, D], k / v [B, Lk, heads_k, D] (dtype N3D_F16 or N3D_BF16; element strides (batch, token, head), multiples of 8, dense
 * channels; 16-byte aligned; D a multiple of 8 up to 128; heads_q a multiple of heads_k: query head h reads key head h / (heads_q / heads_k)) ->
 * out [B, Lq, heads_q, D] dense, lse [B, heads_q, Lq] float32 (logarithm of the softmax's sum; may be NULL; needed for the gradient).
 * With n = lengths[b] (NULL: Lk) keys in use, query i stands at position i + n - Lq (the last query beside the last key):
 *   t = scale * q.k;   softcap > 0: t = softcap * tanh(t / softcap);   slopes [heads_q] float32: t -= slope * |position - j|
 *   visible: j < n; causal: j <= position or j < prefix[b] (prefix [B] int32 or NULL); documents (int32, [B, Lq] / [B, Lk] with the given batch strides,
 *   both or neither NULL): equal and not negative.
 * A row that sees nothing gives out 0 and lse -inf.  Keys behind n are not read.  float32 softmax and accumulation.
 * Refused: 2^24 blocks of rows (128 queries of a head; up to 24 queries, 32 of the queries and heads of a key head) or more; half of that in the backward pass
 * beyond 96 channels.
 * workspace: n3d_attention_workspace(desc) bytes (-1: refused, see n3d_last_error), 16-byte aligned; nothing in it outlives the call. */
typedef struct {
    const void *q, *k, *v;
    void *out, *out_rest;           /* out_rest: what rounding out to dtype left over, again in dtype, or NULL; given back to n3d_attention_bwd it keeps
                                       sum(dout * out), from which every gradient subtracts, accurate (it may be NULL there too) */
    float* lse;
    const int *prefix, *lengths, *q_documents, *k_documents;
    const float* slopes;
    void* workspace;
    const void* dout;               /* gradient of out (n3d_attention_bwd) */
    void *dq, *dk, *dv;             /* gradients, dense like q / k / v; dq, or dk and dv together, may be NULL */
    int64_t q_strides[3], k_strides[3], v_strides[3], dout_strides[3], q_doc_stride, k_doc_stride, workspace_bytes;
    float scale, softcap;
    int B, Lq, Lk, heads_q, heads_k, D, dtype, causal;
} n3d_attention_desc;
int64_t n3d_attention_workspace(const n3d_attention_desc* desc);
int n3d_attention(const n3d_attention_desc* desc, n3d_stream_t stream);
/* Gradients from the forward call's q, k, v, out and lse and from dout.  dk / dv are summed over the query heads of a key head, in a fixed order: the
 * results are bitwise reproducible.  Rows that see nothing and keys that nobody sees get zeros. */
int64_t n3d_attention_bwd_workspace(const n3d_attention_desc* desc);
int n3d_attention_bwd(const n3d_attention_desc* desc, n3d_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* N3D_H_ */
