/*
 * katsu_cuda.h -- C ABI of libkatsu_cuda.so, the sm_100a replacement for
 * katsu-core's dense CPU loops.
 *
 * The reference (pure Rust, crates/katsu-core) has no FFI of its own; these
 * are the entry points a `katsu-cuda` sys-crate binds with an `extern "C"`
 * block so that the arithmetic call sites of katsu-core can be redirected to
 * the GPU.  Each declaration cites the reference lines it stands in for.
 *
 * Conventions
 *  - every function returns an int32_t status (KATSU_OK == 0); nothing throws,
 *    aborts or prints.  katsu_cuda_last_error_string() describes the most
 *    recent failure on the calling thread.
 *  - all tensors are contiguous row-major f32 (the 8-bit matrices of the integer
 *    product and lists of tokens apart); device pointers come from katsu_cuda_alloc (or any
 *    cudaMalloc'ed memory on the context's device).
 *  - sizes are size_t like the reference's usize; the caller has already run
 *    the reference's shape validation (Geometry::new, matmul rank checks);
 *    the library re-checks what it needs and never launches on bad input.
 *  - one context == one device == one stream; calls are asynchronous on that
 *    stream and ordered with each other; katsu_cuda_sync / katsu_cuda_d2h wait.
 *  - one host thread drives a context (the reference's Tensor is Rc-based and
 *    !Send, crates/katsu-core/src/tensor.rs:95-99).
 */
#ifndef KATSU_CUDA_H
#define KATSU_CUDA_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define KATSU_OK 0
#define KATSU_ERR_INVALID_ARG 1  /* null pointer, zero stride, inconsistent sizes */
#define KATSU_ERR_ALLOC 2        /* device or pinned allocation failed (TensorError::Allocation) */
#define KATSU_ERR_CUDA 3         /* a CUDA runtime call or launch failed */
#define KATSU_ERR_NCCL 4         /* NCCL missing or a collective failed */
#define KATSU_ERR_TIMEOUT 5      /* a bounded device-side wait ran out */
#define KATSU_ERR_NO_DEVICE 6    /* no usable CUDA device / bad ordinal */
#define KATSU_ERR_UNSUPPORTED 7  /* shape outside what the requested kernel handles */

/* Arithmetic modes for the contraction kernels.  FP32 = CUDA-core fma.rn.f32.
 * 3XTF32 = tensor-core split precision (hi*hi + lo*hi + hi*lo into an f32
 * accumulator, 22 significand bits an operand), FP32-grade accuracy.  TF32 =
 * single tensor-core pass (11 bits).  Both take layers of at least 16 channels in
 * multiples of 4, and any shape of 1e6 (matmul: 4e7, in TF32 mode 1.5e7)
 * multiply-adds or more whatever its alignment; smaller ones, low-channel
 * stencils and streaming ops run in f32 on CUDA cores.
 * The parts are fp16 with a power-of-two scale per operand.  An element keeps
 * its 22 (11) bits down to 2^-17 (2^-28) of the operand's largest magnitude and
 * an absolute error of 2^-39 of that magnitude below.  An operand in which 128
 * neighbours of a row, or 16 of a column (the channels of a pixel, the output
 * channels of a weight), all lie below that line is cut into bf16 parts of 24
 * (16) bits instead, with the rest of its call; so is one with infinities or
 * NaNs.  Elements below the line among larger neighbours on both axes keep the
 * absolute error; KATSU_MODE_FP32 has none. */
#define KATSU_MODE_3XTF32 0
#define KATSU_MODE_TF32 1
#define KATSU_MODE_FP32 2

typedef struct katsu_cuda_ctx katsu_cuda_ctx;
typedef struct katsu_cuda_event katsu_cuda_event;

/* ---- context ----------------------------------------------------------- */
int32_t katsu_cuda_device_count(int32_t *out_count);
/* Binds one context to one device ordinal and creates its stream. */
int32_t katsu_cuda_init(int32_t device, katsu_cuda_ctx **out_ctx);
int32_t katsu_cuda_shutdown(katsu_cuda_ctx *ctx);
int32_t katsu_cuda_set_precision(katsu_cuda_ctx *ctx, int32_t mode);
int32_t katsu_cuda_get_precision(katsu_cuda_ctx *ctx, int32_t *out_mode);
const char *katsu_cuda_last_error_string(void);
/* Number of kernels this context has launched so far (for benchmark reports). */
int32_t katsu_cuda_launch_count(katsu_cuda_ctx *ctx, uint64_t *out_count);
/* Raw cudaStream_t of the context, for callers that interleave their own work.  Calls captured from it refer to the
 * context's workspace, as its other calls do: replays wait for these and for each other (the same stream, or events). */
int32_t katsu_cuda_stream(katsu_cuda_ctx *ctx, void **out_stream);

/* ---- memory ------------------------------------------------------------ */
/* Zero-filled device buffer of `count` floats: zeros_buffer,
 * crates/katsu-core/src/tensor.rs:120-125.  count == 0 yields a null pointer.
 * Allocation and release are ordered on the context's stream and served from a
 * cached pool, so a step that frees and re-allocates its buffers does not
 * synchronise the device.  A buffer must be freed through a context whose
 * stream has seen (or been synchronised with) its last use. */
int32_t katsu_cuda_alloc(katsu_cuda_ctx *ctx, size_t count, float **out_ptr);
/* The same without the zeros, for buffers that the next call overwrites. */
int32_t katsu_cuda_alloc_uninit(katsu_cuda_ctx *ctx, size_t count, float **out_ptr);
int32_t katsu_cuda_free(katsu_cuda_ctx *ctx, float *ptr);
int32_t katsu_cuda_zero(katsu_cuda_ctx *ctx, float *dst, size_t count);
/* dst[i] = value: the seed of a backward pass (tensor.rs:309-314) without a host buffer to copy from. */
int32_t katsu_cuda_fill(katsu_cuda_ctx *ctx, float *dst, float value, size_t count);
/* Explicit host<->device transfer for the device storage variant of
 * TensorNode.data (crates/katsu-core/src/tensor.rs:101-107).  d2h waits for the
 * stream (and, like katsu_cuda_sync, returns KATSU_ERR_TIMEOUT when a bounded
 * device-side wait gave up in a kernel before it: the data is then undefined).
 * h2d is ordered on the stream; from pageable memory it returns once the source
 * has been staged, a page-locked source (katsu_cuda_host_alloc) must stay
 * untouched until the next katsu_cuda_sync. */
int32_t katsu_cuda_h2d(katsu_cuda_ctx *ctx, float *dst_device, const float *src_host, size_t count);
int32_t katsu_cuda_d2h(katsu_cuda_ctx *ctx, float *dst_host, const float *src_device, size_t count);
/* d2h without the wait: ordered on the stream, dst_host (page-locked) is valid after the
 * next katsu_cuda_sync.  Lets a caller keep several contexts (streams) of one device busy,
 * e.g. copying one batch chunk out while the next one computes. */
int32_t katsu_cuda_d2h_async(katsu_cuda_ctx *ctx, float *dst_host, const float *src_device, size_t count);
int32_t katsu_cuda_d2d(katsu_cuda_ctx *ctx, float *dst_device, const float *src_device, size_t count);
/* Page-locked host staging buffers so h2d/d2h run at full PCIe rate. */
int32_t katsu_cuda_host_alloc(katsu_cuda_ctx *ctx, size_t count, float **out_ptr);
int32_t katsu_cuda_host_free(katsu_cuda_ctx *ctx, float *ptr);
/* Waits for everything queued on the context.  KATSU_ERR_TIMEOUT (once) when a bounded
 * device-side wait gave up in any kernel since the last synchronising call. */
int32_t katsu_cuda_sync(katsu_cuda_ctx *ctx);

/* ---- Conv2D ------------------------------------------------------------ */
/* y[n,k,oy,ox] = sum_{c,r,s} x[n,c,oy*stride+r-pad,ox*stride+s-pad] * w[k,c,r,s]
 * over the in-range taps.  Replaces the visit closure of Conv2D::forward,
 * crates/katsu-core/src/conv2d.rs:95-103 with 232-262.  x is [N,C,H,W], w is
 * [K,C,R,S], y is [N,K,OH,OW] with OH=(H+2*pad-R)/stride+1 (same for OW) and is
 * fully overwritten. */
int32_t katsu_cuda_conv2d_fwd(katsu_cuda_ctx *ctx, const float *x, const float *w, float *y,
                              size_t n, size_t c, size_t h, size_t wd, size_t k, size_t r, size_t s,
                              size_t stride, size_t pad);
/* dx[xi] (+)= sum g[yi]*w[wi] and dw[wi] (+)= sum g[yi]*x[xi] over the same tap
 * set: one call == one backward_buffers, crates/katsu-core/src/conv2d.rs:269-292
 * (called from Conv2D::backward conv2d.rs:127-133 and the Conv2D VJP arm
 * tensor.rs:374-381).  dx or dw may be null to skip that output.  accumulate
 * != 0 adds the result to the existing contents, which folds in the
 * `pending[parent] += grad` pass of tensor.rs:383-390; dx and dw must not alias
 * each other. */
int32_t katsu_cuda_conv2d_bwd(katsu_cuda_ctx *ctx, const float *x, const float *w, const float *g,
                              float *dx, float *dw,
                              size_t n, size_t c, size_t h, size_t wd, size_t k, size_t r, size_t s,
                              size_t stride, size_t pad, int32_t accumulate);

/* One backward_buffers (conv2d.rs:269-292) whose upstream gradient is gfactor * gscale[0] * g[i]
 * without that product ever being stored: gscale is a device scalar (null: 1).  The VJP of
 * loss = sum(y * y) hands the convolution exactly this, g = y with gfactor = 2 and gscale = the
 * adjoint of the loss (crates/katsu-core/src/tensor.rs:392-417), so the backward pass reads y where
 * it would otherwise write and re-read a gradient of y's size.  dX and dW are linear in the upstream
 * gradient; kernels that support it scale their outputs, others get the scaled gradient written
 * out once internally.  Same aliasing and accumulate rules as katsu_cuda_conv2d_bwd. */
int32_t katsu_cuda_conv2d_bwd_scaled(katsu_cuda_ctx *ctx, const float *x, const float *w, const float *g,
                                     const float *gscale, float gfactor, float *dx, float *dw,
                                     size_t n, size_t c, size_t h, size_t wd, size_t k, size_t r, size_t s,
                                     size_t stride, size_t pad, int32_t accumulate);
/* y = act(conv(x, w) + bias[k]) with act = max(., 0) when relu != 0; bias may be null.  Bias and
 * ReLU are not in the reference yet (docs/roadmap.md:18-26 lists them as the next layer features);
 * here they ride in the convolution kernel's epilogue where it has one, so a layer's activation
 * costs no extra pass over y. */
int32_t katsu_cuda_conv2d_fwd_bias_relu(katsu_cuda_ctx *ctx, const float *x, const float *w, const float *bias,
                                        float *y, size_t n, size_t c, size_t h, size_t wd, size_t k, size_t r,
                                        size_t s, size_t stride, size_t pad, int32_t relu);
/* The layer's input staged once for forward and backward.  Conv2D keeps its input between forward and
 * backward (crates/katsu-core/src/conv2d.rs:104-107, 130-136); the wide-channel kernels of both read x
 * through a channels-innermost copy that each call otherwise writes for itself.  A caller that holds x
 * anyway can hold that copy too:
 *   katsu_cuda_conv2d_staged_floats  *floats = size of the copy for this shape in the context's CURRENT
 *                                    precision mode, 0 when the shape's kernels use none;
 *   katsu_cuda_conv2d_stage          writes it into `staged` (device memory of that many floats);
 *   katsu_cuda_conv2d_fwd_staged     katsu_cuda_conv2d_fwd_bias_relu reading x through x_staged;
 *   katsu_cuda_conv2d_bwd_staged     katsu_cuda_conv2d_bwd_scaled reading x through x_staged (dW).
 * x_staged may be null (the plain calls).  The copy is only valid for the precision mode, x contents and
 * shape it was written for; results are bit-identical to the plain calls. */
int32_t katsu_cuda_conv2d_staged_floats(katsu_cuda_ctx *ctx, size_t n, size_t c, size_t h, size_t wd, size_t k,
                                        size_t r, size_t s, size_t stride, size_t pad, size_t *floats);
int32_t katsu_cuda_conv2d_stage(katsu_cuda_ctx *ctx, const float *x, float *staged, size_t n, size_t c, size_t h,
                                size_t wd);
int32_t katsu_cuda_conv2d_fwd_staged(katsu_cuda_ctx *ctx, const float *x, const float *x_staged, const float *w,
                                     const float *bias, float *y, size_t n, size_t c, size_t h, size_t wd,
                                     size_t k, size_t r, size_t s, size_t stride, size_t pad, int32_t relu);
int32_t katsu_cuda_conv2d_bwd_staged(katsu_cuda_ctx *ctx, const float *x, const float *x_staged, const float *w,
                                     const float *g, const float *gscale, float gfactor, float *dx, float *dw,
                                     size_t n, size_t c, size_t h, size_t wd, size_t k, size_t r, size_t s,
                                     size_t stride, size_t pad, int32_t accumulate);
/* Backward of that epilogue over y_act [n, k, plane]: dg = g where y_act > 0 else 0 (relu != 0;
 * dg may alias g, or be null when only dbias is wanted), dbias[k] (+)= sum over n and the plane of
 * dg (null: skipped).  With relu == 0 the gradient passes through unchanged: pass dg = null and
 * feed g to katsu_cuda_conv2d_bwd. */
int32_t katsu_cuda_bias_relu_bwd(katsu_cuda_ctx *ctx, const float *y_act, const float *g, float *dg, float *dbias,
                                 size_t n, size_t k, size_t plane, int32_t relu, int32_t accumulate_bias);
/* w[i] -= lr * dw[i], the plain SGD update the roadmap names (docs/roadmap.md:21-22), so that a
 * training step's parameters never leave the device. */
int32_t katsu_cuda_sgd_step(katsu_cuda_ctx *ctx, float *w, const float *dw, float lr, size_t count);

/* ---- matmul ------------------------------------------------------------ */
/* c[m,n] = a[m,k] @ b[k,n]; Tensor::matmul, crates/katsu-core/src/tensor.rs:264-273.
 * c is fully overwritten (zero when k == 0). */
int32_t katsu_cuda_matmul_fwd(katsu_cuda_ctx *ctx, const float *a, const float *b, float *c,
                              size_t m, size_t k, size_t n);
/* da[m,k] (+)= g[m,n] @ b^T ; db[k,n] (+)= a^T @ g.  Matmul VJP arm,
 * crates/katsu-core/src/tensor.rs:418-445 (which accumulates into the pending
 * adjoints: pass accumulate != 0 for that behaviour).  da or db may be null.
 * da and db may be the same buffer only when m == k == n and the caller wants
 * the reference's "same parent, both edges" sum (tensor.rs:425-444): the buffer
 * then receives g @ b^T + a^T @ g (added to its contents when accumulate != 0). */
int32_t katsu_cuda_matmul_bwd(katsu_cuda_ctx *ctx, const float *a, const float *b, const float *g,
                              float *da, float *db, size_t m, size_t k, size_t n, int32_t accumulate);

/* ---- norms around a block ------------------------------------------------
 * No counterpart in the reference.  With N(v; w, b) = (v - mean) / sqrt(var + eps) * w + b over the last axis
 * (KATSU_NORM_LAYER; var = mean((v - mean)^2)) or v / sqrt(mean(v^2) + eps) * w + b (KATSU_NORM_RMS), for every
 * row of `cols` values:
 *     r = x + scale * gate * N(h; post)      the residual stream behind a block with output h
 *     n = N(r; pre)                          the input of the next block
 * Parts that are left out:
 *     h null        r = x is not written: only n = N(x; pre); gate, post_w, post_b and r are null
 *     post_w null   h itself in place of N(h; post); post_b is null
 *     gate null     1 in its place (gate_rows 0)
 *     n null        no norm behind the sum; pre_w and pre_b are null
 * post_b and pre_b may be null (no bias).  gate is [gate_rows, cols], gate_rows a divisor of rows: 1 (one value a
 * channel), rows (each row its own), or one row of the gate for every rows / gate_rows rows (sequences of one
 * length).  cols is 1 to 2^30 - 1; without rows nothing is written.  Outputs alias neither inputs nor each other.
 * A row's infinities and NaNs stay in its row.  Sums are f32: squares above the f32 range (values above 1.8e19)
 * overflow to a norm of 0; a row without spread, or of values below 1e-19 only, needs eps > 0. */
#define KATSU_NORM_RMS 0
#define KATSU_NORM_LAYER 1
int32_t katsu_cuda_block_norm_fwd(katsu_cuda_ctx *ctx, const float *x, const float *h, const float *gate,
                                  size_t gate_rows, const float *post_w, const float *post_b, const float *pre_w,
                                  const float *pre_b, float scale, float eps, int32_t kind, float *r, float *n,
                                  size_t rows, size_t cols);
/* Backward.  r is what the forward wrote (x where h is null); dr and dn are the gradients of r and n (dr null:
 * zeros; dn is null exactly where pre_w is).  The statistics of the rows are taken again from r and h.
 *     dx = dr + [gradient through N(r; pre)]        dh = [gradient through the gate and N(h; post)] of dx
 *     dgate [gate_rows, cols], dpost_w, dpost_b, dpre_w, dpre_b [cols]: sums over rows, in an order that the
 *     shape and the buffers' alignment fix; zeros where there are no rows
 * Any output may be null.  `accumulate` is a sum of KATSU_BLOCK_*: those outputs are added to their contents. */
#define KATSU_BLOCK_DX 1
#define KATSU_BLOCK_DH 2
#define KATSU_BLOCK_DGATE 4
#define KATSU_BLOCK_DPOST_W 8
#define KATSU_BLOCK_DPOST_B 16
#define KATSU_BLOCK_DPRE_W 32
#define KATSU_BLOCK_DPRE_B 64
int32_t katsu_cuda_block_norm_bwd(katsu_cuda_ctx *ctx, const float *r, const float *h, const float *gate,
                                  size_t gate_rows, const float *post_w, const float *post_b, const float *pre_w,
                                  float scale, float eps, int32_t kind, const float *dr, const float *dn, float *dx,
                                  float *dh, float *dgate, float *dpost_w, float *dpost_b, float *dpre_w,
                                  float *dpre_b, size_t rows, size_t cols, int32_t accumulate);

/* ---- matrix product in 8-bit integers --------------------------------------
 * For a model that is served: y = x w + bias from weights and rows of x in 8 bits, with one scale for every
 * output channel and one for every row (token).  No counterpart in the reference.
 *     scale = max |v| / 127, rounded to f32;  q = v / scale to the nearest whole number, halves to the even one;
 *     y[i][j] = (sum_p q_x[i][p] q_w[p][j]) * scale_x[i] * scale_w[j] + bias[j]
 * The sum is exact (32-bit integers; k is at most KATSU_INT8_MAX_K), so y differs from the real-number formula
 * by the roundings of its conversion, products and sum to f32 only, and no result depends on the other rows.
 * A row (column of w) of zeros has scale 0; one that holds an infinity or a NaN has a NaN for its scale, and so
 * for its results.
 * A quantised matrix of `rows` rows of k values is int8_t [rows][katsu_cuda_int8_row_bytes], the bytes behind k
 * zero, at a 16-byte aligned address; w [k, n] is kept transposed, one row for an output channel.  Outputs overlap
 * neither inputs nor each other. */
#define KATSU_INT8_MAX_K 133144
/* k rounded up to whole 16-byte units. */
int32_t katsu_cuda_int8_row_bytes(size_t k, size_t *out_bytes);
/* w f32 [k, n] -> q int8_t [n][row bytes], scale f32 [n]; done once. */
int32_t katsu_cuda_int8_quantize_weights(katsu_cuda_ctx *ctx, const float *w, int8_t *q, float *scale, size_t k,
                                         size_t n);
/* x f32 [m, k] -> q int8_t [m][row bytes], scale f32 [m]: for several products of the same x. */
int32_t katsu_cuda_int8_quantize_rows(katsu_cuda_ctx *ctx, const float *x, int8_t *q, float *scale, size_t m,
                                      size_t k);
/* y f32 [m, n] from both matrices quantised; bias [n] may be null. */
int32_t katsu_cuda_int8_matmul(katsu_cuda_ctx *ctx, const int8_t *xq, const float *xs, const int8_t *wq,
                               const float *ws, const float *bias, float *y, size_t m, size_t k, size_t n);
/* y f32 [m, n] from x f32 [m, k], whose rows are quantised on the way: the same bits as katsu_cuda_int8_quantize_rows
 * and katsu_cuda_int8_matmul one after the other. */
int32_t katsu_cuda_int8_linear(katsu_cuda_ctx *ctx, const float *x, const int8_t *wq, const float *ws,
                               const float *bias, float *y, size_t m, size_t k, size_t n);

/* ---- the norm over all gradients, and clipping ------------------------------
 * norm = sqrt of the sum of all squares over `tensors` buffers of counts[i] floats (counts of 0 are fine), summed
 * in 64 bits in an order that counts and alignment fix; norm[0] is f32 device memory apart from them.  The arrays
 * of addresses and counts are host memory, read before the call returns.  No counterpart in the reference. */
int32_t katsu_cuda_grad_norm(katsu_cuda_ctx *ctx, const float *const *grads, const size_t *counts, size_t tensors,
                             float *norm);
/* out[i] = grads[i] * min(1, max_norm / norm); out[i] may be grads[i] itself, other overlaps of an output are
 * refused.  Where norm <= max_norm the values stay as they are, bit for bit; so they do where a gradient is
 * infinite or NaN, which norm[0] then shows.  max_norm is 0 or more. */
int32_t katsu_cuda_clip_grads(katsu_cuda_ctx *ctx, const float *const *grads, float *const *out, const size_t *counts,
                              size_t tensors, float max_norm, float *norm);
/* weights[i] -= lr * (grads[i] * min(1, max_norm / norm)): katsu_cuda_clip_grads and katsu_cuda_sgd_step in one,
 * without the clipped gradients being stored (the same bits; grads stay as they are).  Where a gradient is infinite
 * or NaN no weight changes.  Weights overlap neither gradients nor each other. */
int32_t katsu_cuda_sgd_step_clipped(katsu_cuda_ctx *ctx, float *const *weights, const float *const *grads,
                                    const size_t *counts, size_t tensors, float lr, float max_norm, float *norm);

/* ---- the two ends of a language model -----------------------------------------
 * No counterpart in the reference.  Tokens are int32_t in device memory (katsu_cuda_alloc's 4-byte elements), 0 to
 * vocab - 1; what stands for no token (padding, a list's unused places) is any other number.  vocab and the numbers of
 * tokens and rows are below 2^31.  Outputs overlap neither inputs nor each other unless a function says so.
 *
 * Lookup: y[i] = scale * table[tokens[i]] for `count` tokens and a table [vocab, cols]; a row of zeros where tokens[i]
 * is no token. */
int32_t katsu_cuda_embed_fwd(katsu_cuda_ctx *ctx, const float *table, const int32_t *tokens, float scale, float *y,
                             size_t count, size_t vocab, size_t cols);
/* The same from a table in 8 bits, y[i][j] = (q[tokens[i]][j] * rows_scale[tokens[i]]) * scale: q [vocab][row bytes of
 * cols] and rows_scale [vocab] as katsu_cuda_int8_quantize_weights leaves them for w [cols, vocab] (a head whose weights
 * are the table too), or katsu_cuda_int8_quantize_rows for a table [vocab, cols]. */
int32_t katsu_cuda_int8_embed(katsu_cuda_ctx *ctx, const int8_t *q, const float *rows_scale, const int32_t *tokens,
                              float scale, float *y, size_t count, size_t vocab, size_t cols);
/* Gradient of the lookup's table: dtable[v] = scale * (sum of dy[i] over all i with tokens[i] == v), in an order that
 * the tokens and the sizes alone fix: the same bits every time.  Rows of other tokens are zeros.  accumulate != 0: added to dtable
 * instead, whose other rows are not touched. */
int32_t katsu_cuda_embed_bwd(katsu_cuda_ctx *ctx, const int32_t *tokens, const float *dy, float scale, float *dtable,
                             size_t count, size_t vocab, size_t cols, int32_t accumulate);

/* Loss of logits z [rows, vocab] against a teacher's top logits and against labels, for every row:
 *     p = softmax(teacher / T) over the row's `top` entries, q = softmax(z / T) over the vocabulary (T = temperature, a normal number)
 *     loss = weight * (soft T^2 sum_j p_j (log p_j - log q[index_j]) - hard log softmax(z)[label])
 * teacher and index are [rows, top], top at most KATSU_DISTILL_MAX_TOP.  Entries whose index is no token are left out,
 * and a token that is listed twice has both probabilities.  Without an entry that counts (none listed, all teacher
 * logits -infinity) a row's soft part is 0, without a label its hard part.  labels may be null (none), weight null (1).
 * A row of weight 0 is not read: its loss is 0 and its gradient zeros, as they are without either part.  Other rows keep
 * infinities and NaNs to themselves: a logit of -infinity is a token of probability 0 (the loss is infinite where the teacher or the label asks
 * for it), other infinities and NaNs make the row NaN, and so do -infinities only. */
#define KATSU_DISTILL_MAX_TOP 1024
int32_t katsu_cuda_distill_fwd(katsu_cuda_ctx *ctx, const float *logits, const float *teacher, const int32_t *index,
                               const int32_t *labels, const float *weight, float temperature, float soft, float hard,
                               float *loss, size_t rows, size_t vocab, size_t top);
/* dlogits = g[row] * weight * (soft T (q - p) + hard (softmax(z) - [v == label])): the gradient of sum_row g * loss.
 * g [rows] may be null (1).  loss [rows] may be null; otherwise it receives the loss as well (of long rows to the roundings
 * of another order of sums than the call above takes), so that a training step reads the logits once for both.  dlogits may be `logits` itself; accumulate != 0 adds to dlogits (then not `logits`). */
int32_t katsu_cuda_distill_bwd(katsu_cuda_ctx *ctx, const float *logits, const float *teacher, const int32_t *index,
                               const int32_t *labels, const float *weight, float temperature, float soft, float hard,
                               const float *g, float *loss, float *dlogits, size_t rows, size_t vocab, size_t top,
                               int32_t accumulate);

/* Logits [rows, vocab] of a served model before a token is picked from them; for every row and token, in this order:
 *     repetition   v > 0 ? v / repetition : v * repetition for tokens of the row's history
 *     counts       v - (frequency * count + presence) for tokens that are `count` > 0 times in its generated part
 *     biases       v + the values that the row's list has for the token
 *     allowed      -infinity where the token's bit is 0, whatever v is
 * history [rows, history_cols]: the first lengths[row] entries are the row's tokens (null: all), of which the first
 * prompts[row] are its prompt (null: none) and the rest generated; lengths are cut off at 0 and history_cols, prompts at
 * 0 and the length.  repetition, presence, frequency [rows] may be null (1, 0, 0); history is null with history_cols 0.
 * bias_tokens and bias [rows, biases], at most KATSU_LOGITS_MAX_BIASES (null with biases 0): values of one token are
 * added up first.  allowed: bit v % 32 of word v / 32 of [rows][(vocab + 31) / 32], null: every token.
 * out may be `logits` itself. */
#define KATSU_LOGITS_MAX_BIASES 1024
int32_t katsu_cuda_adjust_logits(katsu_cuda_ctx *ctx, const float *logits, const int32_t *history, const int32_t *prompts,
                                 const int32_t *lengths, const float *repetition, const float *presence,
                                 const float *frequency, const int32_t *bias_tokens, const float *bias,
                                 const uint32_t *allowed, float *out, size_t rows, size_t vocab, size_t history_cols,
                                 size_t biases);

/* ---- streaming ops that keep the autograd graph on the device ---------- */
/* out = a + b / out = a * b; Tensor::elementwise, tensor.rs:226-233. */
int32_t katsu_cuda_add(katsu_cuda_ctx *ctx, const float *a, const float *b, float *out, size_t count);
int32_t katsu_cuda_mul(katsu_cuda_ctx *ctx, const float *a, const float *b, float *out, size_t count);
/* out[0] = sum(a); Tensor::sum, tensor.rs:243-247.  Pairwise/tree order on the
 * device (the reference folds left to right). */
int32_t katsu_cuda_sum(katsu_cuda_ctx *ctx, const float *a, float *out, size_t count);
/* Same result as katsu_cuda_sum for callers that cannot allocate device memory (all of
 * it belongs to the host program's own pool, or the implicit synchronisation of
 * cudaMalloc is unacceptable).  Has no counterpart in the reference.  Its per-block
 * partial sums live in a 16 KiB array inside the library image, held by every GPU that
 * loads the library until exit; it calls no allocating routine.  At most
 * KATSU_SUM_STATIC_MAX_COUNT elements, more is refused with KATSU_ERR_UNSUPPORTED.  The
 * array is shared by all calls on a device and keeps the last call's partials: calls that
 * overlap on the GPU (other contexts or streams of the same device) race; calls through
 * one context are stream-ordered.  The first call on a device resolves the array's
 * address and should come before any stream capture, and before the host program's pool
 * takes the rest of the device memory (the driver may place the library's kernel image on
 * the device at that first use). */
#define KATSU_SUM_STATIC_MAX_COUNT ((size_t)1 << 30)
int32_t katsu_cuda_sum_static(katsu_cuda_ctx *ctx, const float *a, float *out, size_t count);
/* out[0] = sum_i a[i] * a[i]: Tensor::mul(a, a) followed by Tensor::sum (tensor.rs:226-247) in one
 * pass over a, every square rounded to f32 before it is added (as the product tensor would hold
 * it) and the same summation tree as katsu_cuda_sum, so the result equals the two-step one bit for
 * bit while the product tensor is never written. */
int32_t katsu_cuda_sumsq(katsu_cuda_ctx *ctx, const float *a, float *out, size_t count);
/* dst[i] (+)= s[0]*src[i] + s[0]*src[i]: both Mul VJP edges of q = y * y (tensor.rs:392-409) when
 * the adjoint of q is the broadcast of one device scalar s[0] (what the Sum VJP produces,
 * tensor.rs:410-417), without that broadcast being stored. */
int32_t katsu_cuda_square_vjp(katsu_cuda_ctx *ctx, float *dst, const float *src, const float *s, size_t count,
                              int32_t accumulate);
/* dst += g : Add VJP edge (tensor.rs:400-408), adjoint accumulation
 * (tensor.rs:387-389) and gradient publication (tensor.rs:353-356). */
int32_t katsu_cuda_axpy_acc(katsu_cuda_ctx *ctx, float *dst, const float *g, size_t count);
/* dst += g * other : Mul VJP edge, tensor.rs:400-408. */
int32_t katsu_cuda_mul_acc(katsu_cuda_ctx *ctx, float *dst, const float *g, const float *other, size_t count);
/* dst += g[0] : Sum VJP, tensor.rs:410-417. */
int32_t katsu_cuda_bcast_acc(katsu_cuda_ctx *ctx, float *dst, const float *g, size_t count);

/* ---- data-parallel gradient exchange (no counterpart in the reference,
 *      which is single-threaded; batch shards over GPUs and only dW sums) --- */
#define KATSU_COMM_ID_BYTES 128
int32_t katsu_cuda_comm_unique_id(uint8_t out_id[KATSU_COMM_ID_BYTES]);
int32_t katsu_cuda_comm_init(katsu_cuda_ctx *ctx, const uint8_t id[KATSU_COMM_ID_BYTES],
                             int32_t n_ranks, int32_t rank);
int32_t katsu_cuda_comm_destroy(katsu_cuda_ctx *ctx);
/* In-place sum over all ranks of a flat gradient bucket, on the context's stream.  Buckets of up to
 * 64 KiB on ranks that share a machine go through IPC-mapped mailboxes in one kernel per rank (a
 * bounded wait for the peers: a rank that never arrives shows as KATSU_ERR_TIMEOUT at the next
 * synchronising call); everything else is one ncclAllReduce.  Every rank receives the same bits. */
int32_t katsu_cuda_allreduce_sum(katsu_cuda_ctx *ctx, float *buf, size_t count);

/* ---- diagnostics (no counterpart in the reference) ------------------------ */
/* Launches one block that waits, for at most `cycles` SM clocks (1e3..2e8), on a barrier
 * nothing signals.  The wait gives up and the kernel returns; the next synchronising call
 * (katsu_cuda_sync, katsu_cuda_d2h, katsu_cuda_event_elapsed_ms) then returns
 * KATSU_ERR_TIMEOUT once and the context remains usable.  Exercises the bounded-wait path of
 * the pipelined kernels without faulting or hanging the device. */
int32_t katsu_cuda_selftest_wait_timeout(katsu_cuda_ctx *ctx, uint64_t cycles);
/* Runs the mailbox all-reduce with `ranks` (1..16) emulated ranks on this one device: buf holds
 * ranks * count floats (count <= 16384), rank r's bucket at r * count, and every bucket ends up
 * holding the sum.  absent > 0 leaves that many ranks out; the others give up after `cycles` SM
 * clocks (1e3..2e9) and the next synchronising call returns KATSU_ERR_TIMEOUT once. */
int32_t katsu_cuda_selftest_mailbox_allreduce(katsu_cuda_ctx *ctx, float *buf, int32_t ranks, size_t count,
                                              int32_t absent, uint64_t cycles);

/* ---- timing on the context's stream ------------------------------------ */
int32_t katsu_cuda_event_create(katsu_cuda_ctx *ctx, katsu_cuda_event **out_event);
int32_t katsu_cuda_event_record(katsu_cuda_ctx *ctx, katsu_cuda_event *event);
/* Waits for `stop`, then returns the milliseconds between the two records. */
int32_t katsu_cuda_event_elapsed_ms(katsu_cuda_ctx *ctx, katsu_cuda_event *start, katsu_cuda_event *stop,
                                    float *out_ms);
int32_t katsu_cuda_event_destroy(katsu_cuda_ctx *ctx, katsu_cuda_event *event);
/* Makes the work queued on `ctx` after this call wait, on the device, for everything that was
 * queued before `event` was last recorded (on this or another context of the same device).
 * The host does not block.  No counterpart in the reference (it has one thread and no queue);
 * it lets two contexts pipeline batch chunks without a host synchronisation per step. */
int32_t katsu_cuda_wait_event(katsu_cuda_ctx *ctx, katsu_cuda_event *event);
/* Overwrites a private buffer larger than L2 so the next kernel starts cold. */
int32_t katsu_cuda_flush_l2(katsu_cuda_ctx *ctx);

#ifdef __cplusplus
}
#endif
#endif /* KATSU_CUDA_H */
