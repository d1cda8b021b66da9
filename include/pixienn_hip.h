/*
 * pixienn_hip.h -- C ABI of the MI355X (gfx950) non-convolution layer kernels.
 *
 * Drop-in boundary for PixieNN's kernel entry points (the free functions the
 * reference declares in its include/<Name>.cuh headers and calls from the layers
 * under include/cuda/).
 * Each function cites the reference interface it replaces as <file>:<lines>.
 *
 * Conventions
 *   - every pointer is a DEVICE pointer unless its name starts with "host_";
 *     tensors are fp32, NCHW, contiguous: index = ((n*C + c)*H + y)*W + x;
 *   - `stream` is a hipStream_t passed as void* (NULL = the default stream);
 *     no function synchronises the device, callers order work through the
 *     stream (the reference's cudaDeviceSynchronize() calls are not kept);
 *   - return value: PXH_OK (0); PXH_ERR_* (< 0) for a rejected call, nothing
 *     was launched; > 0 is the hipError_t of a failed launch.
 *     pxh_last_error() gives the message of the calling thread's last failure;
 *   - buffers are caller owned.  Aliasing is only allowed where a function
 *     says so ("in place").
 */
#ifndef PIXIENN_HIP_H
#define PIXIENN_HIP_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

#define PXH_OK 0
#define PXH_ERR_INVALID_ARGUMENT (-1)
#define PXH_ERR_UNSUPPORTED (-2)
#define PXH_ERR_WORKSPACE (-3)

/* include/ActivationTypes.h:19-30 (same numbering) */
enum pxh_activation {
    PXH_LEAKY = 0, PXH_LINEAR, PXH_LOGGY, PXH_LOGISTIC, PXH_MISH,
    PXH_RELU, PXH_SOFTPLUS, PXH_SWISH, PXH_TANH
};

/* Types of values in memory, where an entry point takes `type` and void pointers: fp32, bfloat16, IEEE half, and the
 * 8-bit e4m3 (4 exponent bits with bias 7, 3 mantissa bits, no infinities, largest value 448). */
enum pxh_type { PXH_F32 = 0, PXH_BF16, PXH_F16, PXH_E4M3 };

const char* pxh_last_error(void);
/* library version, bumped when a signature changes or a declaration leaves this header
 * (2: the test hooks moved to a private header; the tensor tables, the norm-from-the-writer entry
 * points, pxh_reserve_workspace and pxh_bn_train_act_forward_static were added) */
int pxh_abi_version(void);

/* Entry points that take `(workspace, workspace_bytes)` use a per-device buffer owned by the library
 * when given NULL.  That buffer grows when a call needs more than it holds, which allocates device
 * memory and is therefore refused (PXH_ERR_WORKSPACE) while the call's stream is being captured into a
 * graph.  pxh_reserve_workspace makes the current device's buffer hold at least `bytes` (the largest
 * *_workspace_bytes() of the calls to come) ahead of time -- it allocates, so it is a call for BEFORE a
 * capture, not inside one; when the buffer grows it at least doubles, and blocks handed out earlier stay
 * allocated, so addresses that queued work or captured graphs hold remain valid (what is left behind adds
 * up to less than the live block).  The buffer is shared by every
 * NULL-workspace call on the device: calls that may overlap (several streams or threads) must pass
 * workspaces of their own.  No counterpart in the reference (cuDNN and cuBLAS own their scratch). */
int pxh_reserve_workspace(size_t bytes);

/* ------------------------------------------------------------------------
 * Conv-layer epilogue, forward.
 * ---------------------------------------------------------------------- */

/* BN-inference + activation in one pass:
 *   y = act( ((x - rolling_mean[c]) / (sqrt(rolling_var[c]) + 1e-5)) * scale[c] + bias[c] )
 * with the rounding sequence of the CPU layer (subtract, divide, scale, add
 * each rounded to fp32).  pre_activation (nullable) receives the value before
 * act.  In place allowed (y == x).
 * Two launches: the per-channel constants are folded into `workspace`
 * (pxh_bn_folded_bytes(channels) bytes, or NULL for the library's per-device buffer), then the
 * tensor is streamed once.
 * Replaces, for an inferring ConvLayer/BatchNormLayer: cudnnBatchNormalizationForwardInference
 * + preActivation_.copy + activate(), include/cuda/ConvLayer.h:284-307; CPU semantics
 * src/BatchNorm.cpp:24-67 (training == false), include/ConvLayer.h:227-236. */
int pxh_bn_infer_act_forward(const float* x, float* y, float* pre_activation,
                             const float* rolling_mean, const float* rolling_var,
                             const float* scale, const float* bias,
                             int batch, int channels, int spatial, int activation,
                             void* workspace, size_t workspace_bytes, void* stream);

/* The same, split for a layer whose weights do not change between calls: fold once (after
 * loading or updating the weights), then every forward is the single streaming launch.
 * `folded` is a caller-owned, 16-byte aligned device buffer of pxh_bn_folded_bytes(channels).
 * No counterpart in the reference, whose cuDNN call re-derives the constants on every forward. */
size_t pxh_bn_folded_bytes(int channels);
int pxh_bn_fold(const float* rolling_mean, const float* rolling_var, const float* scale,
                const float* bias, int channels, void* folded, void* stream);
int pxh_bn_folded_act_forward(const float* x, float* y, float* pre_activation, const void* folded,
                              int batch, int channels, int spatial, int activation, void* stream);

/* bias + activation in one pass: y = act(x + bias[c]); pre_activation nullable; in place allowed.
 * Replaces addBiasGpu (include/BiasKernels.cuh:21) + preActivation_.copy + activate()
 * (include/Activation.cuh:26) for a ConvLayer without batch_normalize. */
int pxh_bias_act_forward(const float* x, float* y, float* pre_activation, const float* bias,
                         int batch, int channels, int spatial, int activation, void* stream);

/* Bytes of device workspace that serve the BN training entry points for this shape and for every shape with no
 * more images, channels or values per plane. */
size_t pxh_bn_workspace_bytes(int batch, int channels, int spatial);

/* BN-training forward + activation:
 *   mean[c], var[c] (population variance) over N*H*W; rolling = 0.99*rolling + 0.01*stat;
 *   x_hat = (x - mean)/(sqrt(var) + 1e-5); pre = x_hat*scale + bias; y = act(pre).
 * Outputs x_saved, x_norm, pre_activation are each nullable (not materialised when NULL);
 * y == x is allowed when x_saved is NULL or distinct from x.
 * workspace: pxh_bn_workspace_bytes() bytes, or NULL to use a per-device buffer the
 * library allocates on first use and keeps.
 * Replaces cudnnBatchNormalizationForwardTraining + the x_/preActivation_ copies + activate(),
 * include/cuda/ConvLayer.h:284-307, include/cuda/BatchNormLayer.h:59-92; CPU semantics
 * src/BatchNorm.cpp:47-66, src/CpuUtil.cpp:248-301. */
int pxh_bn_train_act_forward(const float* x, float* y, float* pre_activation, float* x_saved,
                             float* x_norm, float* mean, float* var, float* rolling_mean,
                             float* rolling_var, const float* scale, const float* bias,
                             int batch, int channels, int spatial, int activation,
                             void* workspace, size_t workspace_bytes, void* stream);

/* A convolution's epilogue with the ShortcutLayer that follows it in the same pass, for a shortcut with
 * a linear activation over tensors of one shape (every residual block of the shipped YOLOv3 graphs):
 *   y = alpha * act(pre) + beta * from      (two products and one sum, each rounded)
 * i.e. what pxh_shortcut_forward(in = the epilogue's result, from, out = y, alpha, beta, PXH_LINEAR) would
 * leave, without the epilogue's result ever reaching memory: the shortcut's pass (12 bytes per element)
 * becomes one more stream read by the epilogue (4).  Everything else -- statistics, rolling averages,
 * x_saved, x_norm, pre_activation (the CONVOLUTION's pre-activation) -- as in the call without the
 * shortcut.  `from` may be y itself (read before it is written, element by element) but no other output.
 * The layer's own output is not materialised: only for a layer whose output nothing but the shortcut
 * reads (a route or a second shortcut that names the convolution needs the two separate calls), and
 * the layer's backward must not need its output (pxh_bn_act_backward recomputes from x).  In the
 * backward pass the convolution's delta is alpha times the shortcut's.
 * Replaces include/cuda/ConvLayer.h:284-307 followed by include/cuda/ShortcutLayer.h:23-37. */
int pxh_bn_train_act_shortcut_forward(const float* x, float* y, float* pre_activation, float* x_saved,
                                      float* x_norm, float* mean, float* var, float* rolling_mean,
                                      float* rolling_var, const float* scale, const float* bias,
                                      const float* from, float alpha, float beta, int batch, int channels,
                                      int spatial, int activation, void* workspace, size_t workspace_bytes,
                                      void* stream);
/* The same for inference, on constants folded by pxh_bn_fold (pxh_bn_folded_act_forward + shortcut). */
int pxh_bn_folded_act_shortcut_forward(const float* x, float* y, float* pre_activation, const void* folded,
                                       const float* from, float alpha, float beta, int batch, int channels,
                                       int spatial, int activation, void* stream);

/* A convolution's inference epilogue with the MaxPoolLayer that follows it in the same pass, for the
 * 2 x 2 window at stride 2 over planes of even height and width (five of the six pools of YOLOv3-tiny):
 *   pooled[n][c][i][j] = max over the window of act(bn(x)), compared in the pool's own order
 * i.e. what pxh_bn_folded_act_forward followed by pxh_maxpool_forward (kernel 2, stride 2, padding 1)
 * leaves in the pool's output, to the bit, without the layer's output reaching memory and without the
 * indexes, which only a backward pass reads: 5 bytes per element of x instead of 8 + 6.
 *   y       nullable: the layer's own output, for a layer that something else reads as well (a route);
 *   pooled  batch x channels x height/2 x width/2.
 * PXH_ERR_UNSUPPORTED for an odd height or width, or for tensors off a 16-byte boundary: take the two calls.
 * Replaces include/cuda/ConvLayer.h:284-307 (inference) followed by include/cuda/MaxPoolLayer.h:23-37. */
int pxh_bn_folded_act_maxpool_forward(const float* x, float* y, float* pooled, const void* folded, int batch,
                                      int channels, int height, int width, int activation, void* stream);

/* pxh_bn_train_act_forward for callers that cannot allocate device memory and have no workspace
 * to pass (code under HIP graph capture, serving loops, harnesses that forbid hipMalloc): same
 * arguments without the workspace, same kernels, same results.  The partial sums and per-channel
 * constants go into a buffer of PXH_BN_STATIC_SCRATCH_BYTES built into the library's device code
 * (each GPU holds its copy until the process ends); the call allocates and frees nothing.  A shape
 * for which pxh_bn_workspace_bytes() exceeds that size is rejected with PXH_ERR_WORKSPACE before
 * anything is launched.  All calls on one GPU share the buffer: two that overlap in time (different
 * streams or threads) race; order them, or use the workspace form.  The first call on a device looks
 * up the buffer's address, make it outside a capture.
 * No counterpart in the reference (its cuDNN calls own their scratch). */
#define PXH_BN_STATIC_SCRATCH_BYTES ((size_t) 1 << 20)
int pxh_bn_train_act_forward_static(const float* x, float* y, float* pre_activation, float* x_saved,
                                    float* x_norm, float* mean, float* var, float* rolling_mean,
                                    float* rolling_var, const float* scale, const float* bias,
                                    int batch, int channels, int spatial, int activation, void* stream);

/* Per-channel batch statistics only (first half of the above). */
int pxh_bn_stats(const float* x, float* mean, float* var, int batch, int channels, int spatial,
                 void* workspace, size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------
 * Conv-layer epilogue, backward.
 * ---------------------------------------------------------------------- */

/* Activation gradient + BN backward:
 *   d' = delta * act'(pre);  bias_updates[c] += sum d';  scale_updates[c] += sum d' * x_hat;
 *   d'' = d' * scale[c];  mean_delta, var_delta as src/CpuUtil.cpp:303-327;
 *   delta <- d''/sqrt(var+1e-5) + var_delta*2*(x-mean)/(N*HW) + mean_delta/(N*HW)   (in place)
 * x is the saved conv output (x_saved of the forward).  pre_activation may be NULL: it is then
 * recomputed from x exactly as the forward computed it.  mean_delta / var_delta are outputs
 * (nullable).  workspace as for the forward.  Over large slices the workgroups of a channel wait for each other's sums (up to
 * eight such calls may run at once on the units of their streams, beside work that ends by itself); a wait that is starved
 * for seconds ends, and what could not be formed is then NaN.
 * Replaces gradient() + cudnnBatchNormalizationBackward, include/cuda/ConvLayer.h:315-338;
 * CPU semantics include/ConvLayer.h:244-252, src/BatchNorm.cpp:69-96. */
int pxh_bn_act_backward(float* delta, const float* x, const float* pre_activation,
                        const float* mean, const float* var, const float* scale, const float* bias,
                        float* scale_updates, float* bias_updates, float* mean_delta, float* var_delta,
                        int batch, int channels, int spatial, int activation,
                        void* workspace, size_t workspace_bytes, void* stream);

/* Activation gradient + bias backward for a ConvLayer without batch_normalize:
 *   delta *= act'(pre) (in place);  bias_updates[c] += sum over N*HW of delta.
 * Replaces gradient() (include/Activation.cuh:27) + backwardBiasGpu (include/BiasKernels.cuh:22). */
int pxh_bias_act_backward(float* delta, const float* pre_activation, float* bias_updates,
                          int batch, int channels, int spatial, int activation,
                          void* workspace, size_t workspace_bytes, void* stream);

/* Layer::backward's gradient rescale + clip (include/Layer.h:385-397: scaleTensor when the norm of
 * the delta is beyond `threshold`, then clipDelta at +-`clip`; either is off when its figure is <= 0)
 * and the ConvLayer::backward epilogue that follows it (include/ConvLayer.h:238-252) in one call:
 * the same results as pxh_rescale_clip(delta, ...) followed by pxh_bn_act_backward(delta, ...), but the
 * delta is not read once just for its norm -- the first pass of the backward carries the sum of
 * squares and the largest magnitude, the decision is taken on the device, and when nothing has to
 * change (the usual case with the shipped thresholds) the call costs what pxh_bn_act_backward
 * costs plus launches that leave at once.  *norm_out (nullable, device) receives the norm of the
 * delta as it came.  When the delta is rescaled and the clamp moves nothing (in the one-launch
 * backward: nothing in a channel), the sums are not formed again from the rounded factor * delta: they
 * are linear in the delta and are multiplied by the factor instead -- within rounding of the two-call
 * sequence, not bit-identical to it.  When nothing changes the results are those of
 * pxh_bn_act_backward to the bit.
 * workspace: pxh_bn_clipped_workspace_bytes() (enough, like the plain one, for every smaller shape too), or
 * NULL for the library's. */
size_t pxh_bn_clipped_workspace_bytes(int batch, int channels, int spatial);
int pxh_bn_act_backward_clipped(float* delta, const float* x, const float* pre_activation,
                                const float* mean, const float* var, const float* scale, const float* bias,
                                float* scale_updates, float* bias_updates, float* mean_delta, float* var_delta,
                                int batch, int channels, int spatial, int activation,
                                float threshold, float clip, float* norm_out,
                                void* workspace, size_t workspace_bytes, void* stream);

/* The same in front of pxh_bias_act_backward (a ConvLayer without batch_normalize): delta is left
 * rescaled, clamped and multiplied by act'(pre), as the two calls leave it; with a linear activation
 * and nothing to change it is only read.  workspace: pxh_bn_clipped_workspace_bytes(). */
int pxh_bias_act_backward_clipped(float* delta, const float* pre_activation, float* bias_updates,
                                  int batch, int channels, int spatial, int activation,
                                  float threshold, float clip, float* norm_out,
                                  void* workspace, size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------
 * Stand-alone pieces with the reference's own signatures.
 * ---------------------------------------------------------------------- */

/* include/Activation.cuh:26-27 */
int pxh_activate(int activation, float* x, size_t n, void* stream);
int pxh_gradient(int activation, const float* x, size_t n, float* delta, void* stream);
/* include/BiasKernels.cuh:21-22 (bias_updates accumulates) */
int pxh_add_bias(float* output, const float* bias, int batch, int n, int size, void* stream);
int pxh_backward_bias(float* bias_updates, const float* delta, int batch, int n, int size,
                      void* workspace, size_t workspace_bytes, void* stream);
/* include/CudaUtils.cuh:27-31 */
int pxh_fill_f32(float* x, size_t n, float value, void* stream);
/* pxh_fill_f32 for many tensors in a few launches (x, n: HOST arrays of `count` device pointers and
 * element counts): the deltas of all layers, which Layer::forward clears one by one
 * (include/Layer.h:378-383), at the start of a pass. */
int pxh_fill_f32_multi(int count, float* const* x, const size_t* n, float value, void* stream);
int pxh_fill_i32(int* x, size_t n, int value, void* stream);
int pxh_constrain(int n, float alpha, float* x, void* stream);
int pxh_mul(int n, const float* x, float* y, void* stream);          /* y[i] = x[i]*y[i]; x == y allowed */
/* cublasSaxpy as used for "grad += delta", include/cuda/YoloLayer.h:163, cuda/ShortcutLayer.h:49 */
int pxh_axpy(size_t n, float alpha, const float* x, float* y, void* stream);

/* ------------------------------------------------------------------------
 * Route (channel concatenation).  CPU semantics include/RouteLayer.h:91-137 (cblas_scopy /
 * cblas_saxpy per image), device path include/cuda/RouteLayer.h:23-71 (one cudaMemcpy or
 * cublasSaxpy per image and source layer; here one launch per source layer).
 * Image b of the source layer (layer_outputs floats, packed) corresponds to
 * route + b*route_outputs + offset.  forward copies the layer's output into the route's output;
 * backward adds the route's delta slice into the layer's delta.  batch*route_outputs < 2^31.
 * ---------------------------------------------------------------------- */
int pxh_route_forward(const float* layer_output, float* route_output, int batch, int layer_outputs,
                      int route_outputs, int offset, void* stream);
int pxh_route_backward(const float* route_delta, float* layer_delta, int batch, int layer_outputs,
                       int route_outputs, int offset, void* stream);

/* ------------------------------------------------------------------------
 * Max-pool.  include/MaxPoolKernels.cuh:5-7, CPU semantics include/MaxPoolLayer.h:88-158.
 * ---------------------------------------------------------------------- */

/* Writes every element of out and indexes (no prior zero fill needed).  indexes hold the flat
 * NCHW input index of the first strict maximum in row-major window order, or -1. */
int pxh_maxpool_forward(const float* in, float* out, int* indexes, int batch, int channels,
                        int ih, int iw, int oh, int ow, int kernel, int stride, int padding,
                        void* stream);
/* grad[indexes[i]] += delta[i] in ascending i order for every input cell, i.e. bit-identical to
 * the sequential CPU loop also when windows overlap (stride < kernel).  No atomics. */
int pxh_maxpool_backward(const float* delta, const int* indexes, float* grad, int batch, int channels,
                         int ih, int iw, int oh, int ow, int kernel, int stride, int padding,
                         void* stream);
/* The reference's geometry-free signature (maxPoolBackwardGpu).  Float atomics: bit-exact only
 * when no two outputs share an index (stride >= kernel). */
int pxh_maxpool_backward_scatter(const float* delta, const int* indexes, float* grad, int size,
                                 void* stream);

/* ------------------------------------------------------------------------
 * Upsample.  include/UpsampleKernels.cuh:21-22, CPU semantics include/UpsampleLayer.h:97-121.
 * forward != 0: out[b,k,j,i] = scale * in[b,k,j/stride,i/stride]   (plain store, every element)
 * forward == 0: acc[in] += scale * out[...] for the stride^2 covered cells in raster order.
 * ---------------------------------------------------------------------- */
int pxh_upsample(const float* in, int w, int h, int c, int batch, int stride, int forward,
                 float scale, float* acc, float* out, void* stream);
/* The same with the large tensor (`out`) being a channel slice of a wider one: image n of it starts at
 * out + n * out_image_stride (elements, >= c*h*w*stride^2).  With `out` pointing at a channel offset
 * inside the buffer of the route layer that follows (include/RouteLayer.h:91-137), the upsampled
 * tensor lands directly in the concatenation and the route copy of this source is not needed;
 * backward reads the route's delta slice in place. */
int pxh_upsample_strided(const float* in, int w, int h, int c, int batch, int stride, int forward,
                         float scale, float* acc, float* out, long long out_image_stride,
                         void* stream);

/* ------------------------------------------------------------------------
 * Shortcut.  include/ShortcutKernel.cuh:21-22, CPU semantics include/ShortcutLayer.h:84-141.
 * ---------------------------------------------------------------------- */

/* The reference's index-mapped blend: out[oi] = s1*out[oi] + s2*add[ai]. */
int pxh_shortcut(int batch, int w1, int h1, int c1, const float* add, int w2, int h2, int c2,
                 float s1, float s2, float* out, void* stream);
/* Whole ShortcutLayer::forward in one pass (same-shape operands):
 *   pre = alpha*input + beta*from_output; output = act(pre); pre_activation nullable. */
int pxh_shortcut_forward(const float* input, const float* from_output, float* output,
                         float* pre_activation, size_t n, float alpha, float beta, int activation,
                         void* stream);
/* Whole ShortcutLayer::backward in one pass:
 *   delta *= act'(pre_activation) (in place; skipped for linear, pre_activation may then be NULL);
 *   from_delta = 1*from_delta + beta*delta;  grad += alpha*delta (grad nullable). */
int pxh_shortcut_backward(float* delta, const float* pre_activation, float* from_delta, float* grad,
                          size_t n, float alpha, float beta, int activation, void* stream);
/* The same for the call that is the FIRST in a backward pass to write both targets: they are
 * overwritten (from_delta = beta*delta', grad = alpha*delta') instead of accumulated into, which is
 * what accumulating into cleared tensors gives (up to the sign of a zero), so neither needs the
 * zero-fill of Layer::forward (include/Layer.h:378-383) and neither is read: 12 B per element
 * instead of 20 + 8.  In a residual block the shortcut is that call for the delta of the layer in
 * front of it and of its `from` layer (the only other reader of the latter comes earlier in the
 * network, so later in the backward pass).  No counterpart in the reference, which always clears
 * and accumulates; the caller vouches for the order. */
int pxh_shortcut_backward_first(float* delta, const float* pre_activation, float* from_delta,
                                float* grad, size_t n, float alpha, float beta, int activation,
                                void* stream);

/* ------------------------------------------------------------------------
 * YOLO head.  include/YoloKernels.cuh:7-17, CPU semantics include/YoloLayer.h:164-239, 390-547.
 * Layout: [batch][mask][5+classes][area]; entries 0..3 box, 4 objectness, 5.. classes.
 * truths: [batch][max_truth][5] = x, y, w, h, class id (as float); truth_counts[batch].
 * stats[12] (accumulated into, as the reference does): 0 sum IoU, 1 #IoU>.5, 2 #IoU>.75,
 *   3 sum class prob, 4 sum obj at positives, 5 sum obj over all slots, 6 count, 7 class count;
 *   8 box, 9 object, 10 no-object, 11 class sum of squared delta (overwritten).
 * ---------------------------------------------------------------------- */

/* yoloActivateGpu: logistic on entries 0, 1, 4.., copy of entries 2, 3.  In place allowed. */
int pxh_yolo_activate(const float* input, float* output, int batch, int masks, int classes,
                      int area, void* stream);

/* yoloLossGpu with its argument list: region pass over every slot, then the host-assigned
 * positive slots, then cost (sum of squared delta, ADDED to *cost) and loss components.
 * delta must be zero on entry, as in the reference. */
int pxh_yolo_loss(const float* output, float* delta, const float* truths, const int* truth_counts,
                  int max_truth, const int* assigned_classes, const int* assigned_anchors,
                  const float* assigned_boxes, const int* masks, const float* anchors,
                  float* stats, float* cost, int batch, int mask_count, int anchor_count,
                  int classes, int width, int height, int net_width, int net_height,
                  float ignore_thresh, float truth_thresh, float coord_scale, float object_scale,
                  float noobject_scale, float class_scale, void* workspace, size_t workspace_bytes,
                  void* stream);

/* All heads of a model in one pass.  The engine runs each YoloLayer where it sits in the graph
 * (include/Model.h:1740-1759, include/YoloLayer.h:164-239), but nothing reads a head's output delta,
 * cost or statistics before the backward pass: a host that defers its heads to the end of forward
 * hands them over together, and the small heads -- each of which alone is one long chain of dependent
 * steps on a mostly idle machine -- run under the class rows of the large one: two launches for all
 * heads.  Per head the results are those of pxh_yolo_forward_train on that head (output and delta to
 * the bit; the sums are added in another grouping).  Heads share the batch, the truths, the anchor
 * list, the class count and the network size, as the YoloLayers of one model do.
 * masks: host memory; stats[12] / cost[1]: device, nullable.  At most 4 heads per call.
 * workspace: pxh_yolo_heads_workspace_bytes(), or NULL for the library's. */
typedef struct pxh_yolo_head {
    const float* input;
    float* output;
    float* delta;
    const int* masks;
    int mask_count;
    int width, height;
    float ignore_thresh, truth_thresh, coord_scale, object_scale, noobject_scale, class_scale;
    float* stats;
    float* cost;
} pxh_yolo_head;
size_t pxh_yolo_heads_workspace_bytes(int count, const pxh_yolo_head* heads, int batch);
int pxh_yolo_forward_train_heads(int count, const pxh_yolo_head* heads, const float* truths,
                                 const int* truth_counts, int max_truth, const int* host_anchors,
                                 int anchor_count, int batch, int classes, int net_width, int net_height,
                                 void* workspace, size_t workspace_bytes, void* stream);

/* Detections of a decoded head without copying the head to the host: YoloLayer::addDetects
 * (include/YoloLayer.h:601-698) as a thresholded compaction on the device.  A slot passes when its
 * objectness is not below `threshold`; each of its classes with objectness * probability >=
 * threshold gives one record.  image_width/height > 0 selects scaledYoloBox (integer pixel box of
 * the letterboxed image, x/y = left/top), else yoloBox(...).rect() (relative left, top, w, h).
 * *count (device int, cleared by the call) receives the number found, which may exceed `capacity`;
 * only the first `capacity` places are written.  Records are in no particular order; `order` is the
 * position in the reference's emission order (image, cell, mask, class), sort by it to restore it.
 * No counterpart among the reference's device kernels: its CUDA path copies the head to the host. */
typedef struct pxh_detection {
    float x, y, w, h;
    float prob;
    int batch;
    int class_index;
    unsigned order;
} pxh_detection;
int pxh_yolo_detections(const float* predictions, int batch, const int* host_masks, int mask_count,
                        const int* host_anchors, int anchor_count, int classes, int width, int height,
                        int net_width, int net_height, int image_width, int image_height,
                        float threshold, pxh_detection* out, int capacity, int* count, void* stream);
/* The same without clearing *count: the records of this head go behind those already there, and
 * `order_base` is added to their `order` -- with the number of (slot, class) pairs of the heads
 * before it, the orders of a model's heads continue as in Model::detections (include/Model.h:
 * 1078-1088), which asks one YOLO layer after the other. */
int pxh_yolo_detections_append(const float* predictions, int batch, const int* host_masks,
                               int mask_count, const int* host_anchors, int anchor_count, int classes,
                               int width, int height, int net_width, int net_height, int image_width,
                               int image_height, float threshold, unsigned order_base,
                               pxh_detection* out, int capacity, int* count, void* stream);

/* nms (src/Box.cpp:56-147) on records that never leave the device.  The input sequence of the
 * reference is the records' `order` (unique; ties in probability keep it, as its stable sort does).
 * *count (device) says how many of records[capacity] are there (more than capacity = capacity).
 * Records must name images in [0, batch) and classes in [0, classes).  kept[capacity] receives the
 * survivors sorted by descending probability, *kept_count (device) their number.  threshold >= 0.
 * Steps: near-identical boxes (overlap ratio > 0.9) of different classes in one image keep the
 * strongest; then greedy suppression above `threshold` inside each (image, class) group over its
 * first 1024 members.  Workspace: pxh_nms_workspace_bytes(capacity), which serves any batch and every
 * shorter list too, or NULL for the library's.  A capacity of at most 512 (an inference pass) runs as
 * one launch and needs no workspace. */
size_t pxh_nms_workspace_bytes(int capacity);
int pxh_nms(const pxh_detection* records, const int* count, int capacity, int batch, int classes,
            float threshold, pxh_detection* kept, int* kept_count, void* workspace,
            size_t workspace_bytes, void* stream);

size_t pxh_yolo_workspace_bytes(int batch, int mask_count, int classes, int width, int height,
                                int max_truth);

/* Whole YoloLayer::forward of a loss-computing pass in one sweep over the head: decode, dense
 * delta (every element written, no prior fill), positives assigned on the device from the
 * truths with the CPU layer's rule (best anchor over all anchors, later truth overwrites),
 * cost = sum(delta^2) (written to *cost, not divided by batch) and stats[12] (overwritten).
 * host_masks[mask_count], host_anchors[2*anchor_count] are HOST int arrays (layer constants).  * A workspace serves one stream at a time: the one-launch form of the pass counts its workgroups in at
 * device counters kept per workspace address (zero whenever no launch is using them), so two calls that
 * may overlap -- two streams, two threads -- must pass workspaces of their own, and a launch that never
 * completes (a device fault, a destroyed stream) leaves its counters unusable for that address.
 * pxh_yolo_forward_train_heads uses no such counters. */
int pxh_yolo_forward_train(const float* input, float* output, float* delta, const float* truths,
                           const int* truth_counts, int max_truth, const int* host_masks,
                           const int* host_anchors, float* stats, float* cost, int batch,
                           int mask_count, int anchor_count, int classes, int width, int height,
                           int net_width, int net_height, float ignore_thresh, float truth_thresh,
                           float coord_scale, float object_scale, float noobject_scale,
                           float class_scale, void* workspace, size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------
 * SGD with momentum.  The three BLAS calls of ConvLayer::update for one parameter tensor
 * (include/ConvLayer.h:309-321, include/cuda/ConvLayer.h:388-413) in one pass:
 *   if apply_decay d += (-decay*batch)*w;  w += (lr/batch)*d;  d *= momentum.
 * The reference applies the decay to the weights only, not to biases and scales.
 * ---------------------------------------------------------------------- */
int pxh_sgd_update(size_t n, float* w, float* d, int batch, float lr, float momentum, float decay,
                   int apply_decay, void* stream);

/* ... and for every parameter tensor of a model at once, as pxh_adam_update_multi does for Adam
 * (SGD is the optimiser of every shipped preset). */
int pxh_sgd_update_multi(int count, float* const* w, float* const* d, const size_t* n,
                         const int* apply_decay, int batch, float lr, float momentum, float decay,
                         void* stream);

/* ------------------------------------------------------------------------
 * Gradient rescale and clip, the two helpers Layer::backward runs on delta before a layer's own
 * backward (include/Layer.h:385-397, 479-499; include/cuda/Layer.h:24-39: cublasSnrm2 +
 * cublasSscal, then constrainGpu) without the host round trip of the norm:
 *   norm = |x|_2;  if (threshold > 0 && norm > 0 && norm > threshold) x *= threshold/norm;
 *   if (clip > 0) x = clamp(x, -clip, clip).
 * norm_out (nullable, device) receives the norm before rescaling.  When nothing has to change,
 * the tensor is read once and not written.  workspace: pxh_rescale_workspace_bytes() bytes or
 * NULL for the library's per-device buffer.
 * ---------------------------------------------------------------------- */
size_t pxh_rescale_workspace_bytes(void);
int pxh_rescale_clip(float* x, size_t n, float threshold, float clip, float* norm_out,
                     void* workspace, size_t workspace_bytes, void* stream);

/* The same for many tensors in a few launches: Layer::update's hooks pass every update buffer of
 * every layer through these helpers (include/Layer.h:400-411, ConvLayer.h:323-340: weights, biases,
 * scales), each with its own norm.  x and n are HOST arrays of `count` device pointers / element
 * counts; norms, if not NULL, is a DEVICE array of `count` floats that receives each tensor's norm
 * (an empty tensor's entry is left alone).  Every tensor ends up exactly as pxh_rescale_clip leaves
 * it.  Workspace: pxh_rescale_multi_workspace_bytes(), or NULL for the library's. */
size_t pxh_rescale_multi_workspace_bytes(void);
int pxh_rescale_clip_multi(int count, float* const* x, const size_t* n, float threshold, float clip,
                           float* norms, void* workspace, size_t workspace_bytes, void* stream);

/* Norm and largest magnitude from the kernel that writes the delta.  Layer::backward opens with the
 * two helpers above on the layer's own delta (include/Layer.h:385-397), which costs a read of the
 * tensor just for the norm.  Where one of this library's kernels is the LAST to write that delta
 * before its layer's backward -- the convolution in front of a shortcut receives its whole delta
 * from the shortcut's backward (include/ShortcutLayer.h:98-111), the layer in front of a YOLO head
 * from the head's `grad += delta` (include/YoloLayer.h:741-750) -- that kernel can leave behind, per
 * group of 256 values, the sum of squares and the largest magnitude of what it wrote (8 bytes per
 * KiB of tensor), and pxh_rescale_clip_from_groups starts from those instead of reading the tensor.
 * The sums are added in the order pxh_rescale_clip itself adds them: norm, verdict and rewritten
 * tensor are the same to the bit.
 *   groups: device buffer of pxh_norm_groups_bytes(n) bytes, 8-byte aligned, owned by the caller;
 *           it describes the tensor only until the tensor is written again.
 * A tensor that is not 16-byte aligned, or whose length is not a multiple of 4, has no group sums:
 * the producers then leave the buffer alone and pxh_rescale_clip_from_groups reads the tensor, so the
 * pair can be used without looking at the pointer.
 *   pxh_norm_groups               the group sums of a tensor as it is (one read)
 *   pxh_axpy_norm                 pxh_axpy, + the group sums of y
 *   pxh_shortcut_backward_norm    pxh_shortcut_backward (first == 0) or pxh_shortcut_backward_first
 *                                 (first != 0), + the group sums of grad, which is required */
size_t pxh_norm_groups_bytes(size_t n);
int pxh_norm_groups(const float* x, size_t n, void* groups, void* stream);
int pxh_axpy_norm(size_t n, float alpha, const float* x, float* y, void* y_groups, void* stream);
int pxh_shortcut_backward_norm(float* delta, const float* pre_activation, float* from_delta,
                               float* grad, size_t n, float alpha, float beta, int activation,
                               int first, void* grad_groups, void* stream);
int pxh_rescale_clip_from_groups(float* x, size_t n, float threshold, float clip, float* norm_out,
                                 const void* groups, void* workspace, size_t workspace_bytes,
                                 void* stream);

/* A ShortcutLayer's whole backward: Layer::backward's rescale + clip of its delta (include/Layer.h:385-397,
 * 474-499), then the shortcut's own backward (include/ShortcutLayer.h:98-111) --
 *   pxh_rescale_clip(delta, n, threshold, clip, norm_out, ...), then
 *   first ? pxh_shortcut_backward_first(delta, ...) : pxh_shortcut_backward(delta, ...)
 * with the values of that sequence to the bit.  For a first writer (first != 0) with a linear activation
 * over 16-byte aligned tensors of a multiple of four values -- every shortcut of the shipped YOLOv3 graph
 * once its targets are known to be written here first -- the two run as two launches that read the
 * delta once when nothing has to change (the common case: the pass that adds up the norm writes both
 * targets as well, the second launch forms the verdict and leaves; otherwise it rewrites the delta and
 * both targets from it): 8 or 12 bytes per element where the sequence moves 12 or 16.  Every other case
 * runs the sequence itself.  delta must not alias from_delta or grad; grad is nullable.
 * workspace: pxh_rescale_workspace_bytes() bytes or NULL. */
int pxh_shortcut_backward_clipped(float* delta, const float* pre_activation, float* from_delta,
                                  float* grad, size_t n, float alpha, float beta, int activation,
                                  int first, float threshold, float clip, float* norm_out,
                                  void* workspace, size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------
 * Adam.  include/Adam.cuh:21, include/cuda/Adam.h:49-90.
 * ---------------------------------------------------------------------- */

/* adamGpu: x += rate * (m/(1-b1^t)) / (sqrt(v/(1-b2^t)) + eps) */
int pxh_adam(int n, float* x, const float* m, const float* v, float beta1, float beta2, float rate,
             float eps, int t, void* stream);
/* Whole Adam<CUDA>::update in one pass, same per-element operation order:
 *   d *= 1/batch; if apply_decay d += -decay*w; m = b1*m + (1-b1)*d; v = b2*v + (1-b2)*d*d;
 *   w += lr * (m/(1-b1^t)) / (sqrt(v/(1-b2^t)) + eps);  d = 0.
 * (apply_decay == 1: L2 decay folded into the update before the moments, as the reference does.)
 * apply_decay == 2 is the decoupled form, which the reference does not have: the moments are formed from
 * the plain update and the weight also shrinks by lr * decay of its old value,
 *   w = (w + lr * (m/(1-b1^t)) / (sqrt(v/(1-b2^t)) + eps)) + (-(lr * decay)) * w,
 * each operation rounded to fp32.  Other values of apply_decay are rejected.  The many-tensor forms
 * below take the reference's form only. */
int pxh_adam_update(size_t n, float* w, float* d, float* m, float* v, int batch, int t, float lr,
                    float beta1, float beta2, float eps, float decay, int apply_decay, void* stream);

/* The same for every parameter tensor of a model in as few launches as possible (the engine updates
 * its layers one by one, cuda/ConvLayer.h:370-386: three tensors per convolution, most of them a few
 * hundred values).  w, d, m, v and n are HOST arrays of `count` device pointers / element counts;
 * apply_decay is a host array of flags (weights: 1, biases and scales: 0) or NULL for none.  Each
 * element gets exactly what pxh_adam_update gives it.  Tensors of length 0 are skipped. */
int pxh_adam_update_multi(int count, float* const* w, float* const* d, float* const* m,
                          float* const* v, const size_t* n, const int* apply_decay, int batch, int t,
                          float lr, float beta1, float beta2, float eps, float decay, void* stream);

/* ------------------------------------------------------------------------
 * The many-tensor operations over a table kept in device memory: ONE launch for all parameter
 * tensors of a model (two for rescale + clip), where the host-array forms above take one launch per
 * 32 tensors.  A model builds its tables once, after its layers exist (the engine's counterpart
 * would be Model::update, include/Model.h:1772-1792, gathering what ConvLayer::update,
 * include/cuda/ConvLayer.h:370-413, and Layer::update, include/Layer.h:400-411, step one by one).
 *
 * pxh_tensor_table_create: `buffers` is a HOST array of streams * count device pointers, stream after
 * stream (buffers[k * count + i] = buffer k of tensor i); streams = 1 (fill, rescale + clip: x),
 * 2 (SGD: w, d) or 4 (Adam: w, d, m, v); n[count] element counts; apply_decay[count] flags or NULL.
 * Tensors of length 0 are left out; at most 2048 tensors.  Allocates device memory and uploads the
 * table with a blocking copy: call it at set-up, not under graph capture.  The table belongs to the
 * device that was current; destroy it with pxh_tensor_table_destroy.  A table with more buffers per
 * tensor than an operation needs serves it too (an Adam table can be filled or rescaled: buffer 0).
 * Every tensor ends up exactly as the single-tensor call leaves it.  pxh_rescale_clip_table keeps
 * its partial sums inside the table, so two calls on one table must not overlap in time; `norms`
 * (nullable, device) receives one norm per tensor of the table, in table order.
 * No counterpart in the reference.
 * ---------------------------------------------------------------------- */
typedef struct pxh_tensor_table pxh_tensor_table;
int pxh_tensor_table_create(int count, int streams, float* const* buffers, const size_t* n,
                            const int* apply_decay, pxh_tensor_table** table);
void pxh_tensor_table_destroy(pxh_tensor_table* table);
/* tensors in the table (those of length 0 are not counted) */
int pxh_tensor_table_count(const pxh_tensor_table* table);
int pxh_adam_update_table(const pxh_tensor_table* table, int batch, int t, float lr, float beta1,
                          float beta2, float eps, float decay, void* stream);
int pxh_sgd_update_table(const pxh_tensor_table* table, int batch, float lr, float momentum, float decay,
                         void* stream);
int pxh_fill_f32_table(const pxh_tensor_table* table, float value, void* stream);
int pxh_rescale_clip_table(const pxh_tensor_table* table, float threshold, float clip, float* norms,
                           void* stream);

/* ------------------------------------------------------------------------
 * Layers of token models: what stands between the matrix products of a network over tokens.  No counterpart in the
 * reference, whose networks are convolutional; the products are not part of this library.
 *
 * Tensors here are rows of values of one type (pxh_type), the values of a row next to each other and the rows `*_stride`
 * values apart (>= the row's length; 0 rows: nothing to do).  Nothing has to be aligned beyond its own values.  Sums,
 * statistics and intermediate values are fp32; a result is rounded once, to nearest even, when it is stored.  As everywhere in
 * this header what a backward pass leaves is ADDED to the parameters by the optimiser: hand in the gradient of what is to
 * grow (a log likelihood).
 * ---------------------------------------------------------------------- */

/* Root-mean-square norm over the rows, with the residual's addition in front of it:
 *   h = x + residual, rounded to `type` (h = x without one);  rstd = 1 / sqrt(mean(h^2) + eps);  y = h * rstd * weight
 * residual, sum (receives h; only with a residual), scales and rstd are nullable.  weight holds `width` values of
 * weight_type: `type` or PXH_F32.  y_type is `type`, or PXH_E4M3 with scales: `group` consecutive values of a row (128, or 0
 * for the whole row; the last group of a row may be shorter) share
 *   scale = largest |y| of the group / 448 (as a product with 1/448; 2^-126 at least, and finite),  and y holds e4m3(y / scale);
 * scales is [rows][width / group, rounded up], packed.  sum may be x or residual itself, and y (of `type`) may be x or
 * residual, where the strides are the same; nothing else that is written may overlap another tensor.  An infinity in a row makes
 * its rstd 0 and the infinite values NaN, a NaN the whole row NaN, as the formulas have it. */
int pxh_rms_norm_forward(const void* x, const void* residual, void* sum, const void* weight, void* y, float* scales,
                         float* rstd, int type, int weight_type, int y_type, long long rows, int width, long long x_stride,
                         long long residual_stride, long long sum_stride, long long y_stride, int group, float eps,
                         void* stream);

/* Its gradients, from h (the sum if there was a residual) and the forward's rstd:
 *   c = mean(dy * weight * h * rstd) over the row;  dx = rstd * (dy * weight - h * rstd * c) + dsum;
 *   dw (+)= sum over the rows of dy * h * rstd
 * dsum (nullable) is what arrives along the residual stream; dx is then the gradient of x and of the residual alike.  dx may be dy
 * or dsum where the strides are the same.  dw[width] is fp32, overwritten (accumulate == 0) or added to; it is summed in a fixed
 * order.  workspace: pxh_rms_norm_workspace_bytes(rows, width), which serves fewer rows and shorter rows too, or NULL for the
 * library's. */
size_t pxh_rms_norm_workspace_bytes(long long rows, int width);
int pxh_rms_norm_backward(const void* dy, const void* h, const void* weight, const float* rstd, const void* dsum, void* dx,
                          float* dw, int type, int weight_type, long long rows, int width, long long dy_stride,
                          long long h_stride, long long dsum_stride, long long dx_stride, int accumulate, void* workspace,
                          size_t workspace_bytes, void* stream);

/* Log probabilities of given tokens, entropy, and the most probable alternatives, one row of logits per token:
 *   z = scale * logits;  lse = log sum exp z;  logp = z[target] - lse;  entropy = lse - sum softmax(z) * z
 * targets: [rows], int32 (wide_targets == 0) or int64; one outside [0, vocab) gives a logp of 0 (a place at which nothing is to
 * be learned).  targets and logp are given together or not at all; entropy and lse are nullable.  scale > 0.
 * top_logp, top_ids [rows][top]: z - lse of the `top` largest z (at most PXH_MOST_ALTERNATIVES, and vocab) and their indices,
 * descending, among equal ones the lowest index first; top == 0: none.  Like logp, top_logp is formed relative to the row's largest
 * z, and so is right where lse, as an fp32 number, has lost the logarithm beside huge logits.
 * A logit of minus infinity has probability 0, and one of the type's lowest value is a number as any other.  A row of nothing but
 * minus infinities has lse and logp minus infinity, entropy 0 (and NaN for its alternatives, which have no distribution); one with a
 * NaN or plus infinity has NaN in all three, and its NaNs come last among the alternatives.
 * A row's results do not depend on where it lies or on the other rows' values; their last bits do on the number of rows, by which the
 * workgroups of a row are chosen.
 * workspace: pxh_token_logprobs_workspace_bytes(rows, vocab, top), which serves fewer rows, fewer alternatives and smaller
 * vocabularies too, or NULL for the library's (most calls write nothing to it: it is for rows in several parts). */
#define PXH_MOST_ALTERNATIVES 64
size_t pxh_token_logprobs_workspace_bytes(long long rows, int vocab, int top);
int pxh_token_logprobs_forward(const void* logits, const void* targets, float* logp, float* entropy, float* lse,
                               float* top_logp, int* top_ids, int type, int wide_targets, long long rows, int vocab,
                               long long stride, int top, float scale, void* workspace, size_t workspace_bytes, void* stream);

/* The gradient of the logits for gradients of logp and entropy (each nullable: none), from the forward's lse, and its entropy where
 * d_entropy is given:
 *   dlogits[j] = scale * (d_logp * ((j == target) - p[j]) - d_entropy * p[j] * (log p[j] + entropy)),  p = exp(z - lse)
 * A row whose target is outside [0, vocab) has no gradient of logp; a row of nothing but minus infinities has zeros.  dlogits, of the
 * logits' type, may be the logits themselves (with the same stride).  lse is taken as it is, rounded to fp32: its rounding, 2^-24 of
 * |lse|, is in every probability (which matters where all logits of a row are huge, as in a row filled with the type's lowest
 * value; the call below is exact there too). */
int pxh_token_logprobs_backward(const void* logits, const void* targets, const float* lse, const float* entropy,
                                const float* d_logp, const float* d_entropy, void* dlogits, int type, int wide_targets,
                                long long rows, int vocab, long long stride, long long d_stride, float scale, void* stream);

/* Both at once, for gradients that are known before (the weights of the tokens in a mean): what the two calls leave, the logits
 * read once where a workgroup's registers hold a row (up to 163840 logits of 16 bits, half as many of fp32).  logp, entropy and lse
 * are nullable. */
int pxh_token_logprobs_forward_train(const void* logits, const void* targets, const float* d_logp, const float* d_entropy,
                                     void* dlogits, float* logp, float* entropy, float* lse, int type, int wide_targets,
                                     long long rows, int vocab, long long stride, long long d_stride, float scale,
                                     void* stream);

/* Rows of a table by token: y[r] = scale * table[tokens[r]], zeros for a token outside [0, vocab).  tokens: [rows], int32
 * (wide_tokens == 0) or int64.  table and y are of `type`. */
int pxh_embedding_forward(const void* table, const void* tokens, void* y, int type, int wide_tokens, long long rows, int vocab,
                          int width, long long table_stride, long long y_stride, float scale, void* stream);

/* The gradient of the table: d[v] = scale * the sum of dy[r] over the rows r of token v (zeros for a token of no row), or, with
 * accumulate, added to what d holds, of which rows without one are not touched.  d is of `type` or fp32 (d_type).  The rows are
 * sorted by token and added up in fp32 in an order that the tokens alone decide: the same call gives the same bits.  Rows whose
 * token is outside the vocabulary count nothing.  dy and d may not overlap.  workspace: pxh_embedding_workspace_bytes(rows, width),
 * which serves fewer rows and shorter ones too, or NULL for the library's. */
size_t pxh_embedding_workspace_bytes(long long rows, int width);
int pxh_embedding_backward(const void* dy, const void* tokens, void* d, int type, int d_type, int wide_tokens, long long rows,
                           int vocab, int width, long long dy_stride, long long d_stride, float scale, int accumulate,
                           void* workspace, size_t workspace_bytes, void* stream);

/* Layer norm over the rows, with the residual's addition in front of it:
 *   h = x + residual, rounded to `type` (h = x without one);  mean = mean(h);  rstd = 1 / sqrt(mean((h - mean)^2) + eps)
 *   y = (h - mean) * rstd * weight + bias
 * residual, sum (receives h; only with a residual), bias, mean and rstd (each [rows], what the backward pass needs) are nullable.
 * weight and bias hold `width` values of weight_type: `type` or PXH_F32.  sum may be x or residual itself, and y may be x or
 * residual, where the strides are the same; nothing else that is written may overlap another tensor. */
int pxh_layer_norm_forward(const void* x, const void* residual, void* sum, const void* weight, const void* bias, void* y,
                           float* mean, float* rstd, int type, int weight_type, long long rows, int width, long long x_stride,
                           long long residual_stride, long long sum_stride, long long y_stride, float eps, void* stream);

/* Its gradients, from h (the sum if there was a residual) and the forward's mean and rstd:
 *   g = dy * weight;  xhat = (h - mean) * rstd;  dx = rstd * (g - mean(g) - xhat * mean(g * xhat)) + dsum
 *   dw (+)= sum over the rows of dy * xhat;  db (+)= sum over the rows of dy
 * dsum (nullable) is what arrives along the residual stream; dx is then the gradient of x and of the residual alike, and may be dy
 * or dsum where the strides are the same.  dw and db (nullable) are fp32, [width], overwritten (accumulate == 0) or added to, summed
 * in a fixed order.  workspace: pxh_layer_norm_workspace_bytes(rows, width), which serves fewer rows and shorter rows too, or NULL
 * for the library's. */
size_t pxh_layer_norm_workspace_bytes(long long rows, int width);
int pxh_layer_norm_backward(const void* dy, const void* h, const void* weight, const float* mean, const float* rstd,
                            const void* dsum, void* dx, float* dw, float* db, int type, int weight_type, long long rows, int width,
                            long long dy_stride, long long h_stride, long long dsum_stride, long long dx_stride, int accumulate,
                            void* workspace, size_t workspace_bytes, void* stream);

/* A gated linear recurrence over sequences of tokens, channel by channel:
 *   z = 1 / (1 + exp(-update));  h[t] = h[t - 1] + z * (x - h[t - 1]);  y = h, or with a gate (nullable) h * gate / (1 + exp(-gate))
 * x, update, gate and y are [rows][width] of `type`; h is fp32 throughout.  The rows are the tokens of `sequences` sequences, one behind
 * the other: starts[sequences + 1] (device, int32, not descending) says where each begins and the last one ends, or, where it is NULL,
 * all are of rows / sequences tokens.  Rows in front of the first and behind the last sequence are not written.  Where starts descends
 * or leaves the rows, the results are unspecified, but nothing beyond the tensors is touched.
 * state, final (nullable, fp32 [slot_count][width]): a sequence begins with its row of state (zeros without), and leaves what h is behind
 * its last token (without tokens: what it began with) in its row of final, which may be state itself.  slots[sequences] (device, int32)
 * says which row is a sequence's, or, where it is NULL, row s is that of sequence s; one outside [0, slot_count) has no row: the sequence
 * begins with zeros and leaves nothing.  Two sequences may not have the same row.
 * saved (nullable, fp32 [rows / PXH_SCAN_SAVED, rounded up][width]) receives h in front of every PXH_SCAN_SAVED-th row, which is what
 * the backward pass needs.  y may be x, update or gate where the strides are the same.
 * A result depends on its sequence alone up to the last bits of h, which depend on where in the rows the sequence lies, and the same
 * call gives the same bits.  Within a step h is rounded to 2^-23 of the larger of |h| and |x|.  Where h is infinite or no number, it is no
 * number from the next token to the end of the sequence, as the formula has it.
 * workspace: pxh_gated_scan_workspace_bytes(rows, width), which serves fewer rows and shorter rows too, or NULL for the library's. */
#define PXH_SCAN_SAVED 16
size_t pxh_gated_scan_workspace_bytes(long long rows, int width);
int pxh_gated_scan_forward(const void* x, const void* update, const void* gate, void* y, const int* starts, const float* state,
                           float* final, const int* slots, float* saved, int type, long long rows, int width, int sequences,
                           int slot_count, long long x_stride, long long update_stride, long long gate_stride, long long y_stride,
                           void* workspace, size_t workspace_bytes, void* stream);

/* Its gradients, from the forward's inputs and what it saved:
 *   G[t] = dy * g + (1 - z[t + 1]) * G[t + 1], with g = 1 or gate / (1 + exp(-gate)), and behind a sequence's last token its d_final
 *   dx = z G;  dupdate = G (x - h[t - 1]) z (1 - z);  dgate = dy h s (1 + gate (1 - s)), s = 1 / (1 + exp(-gate));  d_state = (1 - z) G
 * of a sequence's first token.  gate and dgate go together.  state: what the forward began with (it may not have been overwritten
 * since).  d_final, d_state (nullable, fp32 [slot_count][width]) are the gradients of final and of state, by the forward's slots;
 * d_state may be d_final.  dx may be dy or x, dupdate update and dgate gate, where the strides are the same. */
int pxh_gated_scan_backward(const void* dy, const void* x, const void* update, const void* gate, const float* saved, void* dx,
                            void* dupdate, void* dgate, const int* starts, const float* state, const float* d_final, float* d_state,
                            const int* slots, int type, long long rows, int width, int sequences, int slot_count,
                            long long dy_stride, long long x_stride, long long update_stride, long long gate_stride,
                            long long dx_stride, long long dupdate_stride, long long dgate_stride, void* workspace,
                            size_t workspace_bytes, void* stream);

/* One new token of each of `rows` sequences, in one launch: as the forward with sequences of one token, the states in place. */
int pxh_gated_scan_step(const void* x, const void* update, const void* gate, void* y, float* state, const int* slots, int type,
                        long long rows, int width, int slot_count, long long x_stride, long long update_stride,
                        long long gate_stride, long long y_stride, void* stream);

/* Beam search: of every item's `beams` beams (at most 64) the `count` best continuations (at most PXH_MOST_ALTERNATIVES), by
 *   score[beam][token] = scores[beam] + scale * logits[beam][token] - log sum exp (scale * logits[beam])
 * descending; of equal ones the lower beam's first, in a beam the larger logit's, then the lower token.  logits: [batch * beams][vocab];
 * scores: [batch][beams], what the beams have come to.  A beam that is ended (nullable, [batch][beams], not 0) has one continuation,
 * end_token with the score that it has.  out_scores, parents (the beams) and tokens are [batch][count].  A score of minus infinity (a
 * masked token, a beam that is not there yet, a sum below the fp32 numbers) and one that is no number (a beam whose logits hold a NaN or plus
 * infinity) are no continuations; the places for which there is none have a score of minus infinity, and -1 for parent and token.  Scores
 * are formed and compared in 64 bits, the logits times the scale too, from sums in fp32, and rounded once.  out_scores may be scores where
 * count is beams.
 * workspace: pxh_beam_select_workspace_bytes(batch, beams, vocab, count), which serves fewer of each too, or NULL for the library's. */
size_t pxh_beam_select_workspace_bytes(int batch, int beams, int vocab, int count);
int pxh_beam_select(const void* logits, const float* scores, const unsigned char* ended, float* out_scores, int* parents,
                    int* tokens, int type, int batch, int beams, int vocab, long long stride, int count, int end_token, float scale,
                    void* workspace, size_t workspace_bytes, void* stream);

/* Tensors with a row for each beam, in the beams' new order, in place: row (item, k) becomes what row (item, parents[item][k]) was.
 * A parent outside [0, beams) leaves the row as it is.  tensors, row_bytes and strides (bytes from row to row) are HOST arrays of
 * `count`: the states of layers, histories of tokens, of any type; one launch for every 32 of them.  The tensors may not overlap. */
int pxh_beam_reorder(int count, void* const* tensors, const long long* row_bytes, const long long* strides, const int* parents,
                     int batch, int beams, void* stream);

/* AdamW over all parameter tensors of a model at once, from a table kept on the device, with states in 32 or in 8 bits and the
 * gradients clipped by their common norm:
 *   norm = |d_scale * d|_2 over all tensors;  f = max_norm > 0 and norm > max_norm ? max_norm / norm : 1
 *   g = d * d_scale * f;  m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g^2
 *   w += lr * (m / (1 - beta1^t)) / (sqrt(v / (1 - beta2^t)) + eps) - lr * decay * w     (the decay where apply_decay says so)
 *   copy = w, rounded to its type
 * beta1 and beta2 are taken in 64 bits (1 - beta is what an fp32 beta has lost).  d is only read (unlike pxh_adam_update's).
 * d_scale: 1 / batch, the inverse of a loss scale, or both.  The norm is summed in 64 bits, in a fixed order; f is formed from it
 * there, and both are rounded to fp32 once.
 *
 * States in 8 bits: m and the SQUARE ROOT of v are e4m3 values with a scale for each 256 of a tensor, its largest magnitude / 448
 * (as a product with 1/448, 2^-126 at least): 2 + 1/32 bytes a value for both.  Each step's results are rounded stochastically, up with the
 * probability of the part cut off: what a step changes of an average over 1000 steps is less than half a unit of such a value, and
 * rounded to nearest it would never change.  A root that is not zero never rounds to zero (the quotient stays bounded).  The
 * random bits come from `seed` (its low 31 bits) and the value's place in the table: another seed every step, the step's number
 * for instance; the same seed gives the same bits.  A state that is no number, NaN or infinite, is kept as the largest value of its
 * block, whose scale is that of the others: what is lost is its own weight.  A step reads the states as they were rounded, and
 * applies its own before they are rounded.
 *
 * norm_out (nullable, device) receives the norm, also when max_norm is 0.  With max_norm > 0 and a norm that is not finite as an fp32
 * number (an overflow of half-precision gradients, or finite ones that are too large together) nothing is written but norm_out: the
 * step is left out.
 *
 * pxh_adamw_table_create copies `tensors` (host memory); those of no values are left out; any number up to 2^20, of less than
 * 2^31 values each.  state_bits is 32 (m, v: floats, the scales null) or 8.  The buffers need the alignment of their own values.
 * Allocates device memory and uploads with a blocking copy: call it at set-up, not under graph capture.  The table belongs to
 * the device that was current, and a step to a current device that is another is refused.  The norm's partial sums lie in the
 * table: two steps of one table must not overlap in time. */
typedef struct pxh_adamw_tensor {
    float* w;
    const void* d;          /* of d_type: PXH_F32, PXH_BF16 or PXH_F16 */
    void* m;
    void* v;
    float* m_scale;         /* 8 bits: [n / 256, rounded up] */
    float* v_scale;
    void* copy;             /* nullable; of copy_type: PXH_BF16 or PXH_F16 */
    size_t n;
    int d_type, copy_type, apply_decay;
} pxh_adamw_tensor;
typedef struct pxh_adamw_table pxh_adamw_table;
int pxh_adamw_table_create(int count, const pxh_adamw_tensor* tensors, int state_bits, pxh_adamw_table** table);
void pxh_adamw_table_destroy(pxh_adamw_table* table);
/* tensors in the table (those of no values are not counted) */
int pxh_adamw_table_count(const pxh_adamw_table* table);
int pxh_adamw_update_table(const pxh_adamw_table* table, int t, float lr, double beta1, double beta2, float eps, float decay,
                           float d_scale, float max_norm, float* norm_out, unsigned seed, void* stream);

#ifdef __cplusplus
}
#endif
#endif
