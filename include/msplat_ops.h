/*
 * msplat_ops.h — C ABI of the operators for learned per-Gaussian attributes.
 *
 * A caller may keep a learned feature vector per Gaussian of a fixed set (the
 * trainer's checkpoints and densification do not carry it). These operators turn
 * such features into what the training step reads or is trained on:
 *   msplat_linear_*              fully connected layers, e.g. the [N,3] colours
 *                                that msplat_shard_forward_backward_rgb takes
 *                                and, from the colour columns of its gradient
 *                                records, their gradients
 *   msplat_dropout               dropout, forward and backward
 *   msplat_loss_cross_entropy    a label loss with its gradients, beside
 *                                msplat_loss_ssim_noalloc
 * Weights of MSPLAT_DTYPE_F32 are updated from their gradients with
 * msplat_fused_adam, which takes that type only.
 * None of them has a counterpart in the reference.
 *
 * Matrices are row-major device memory of the current device with a row
 * stride in elements (ld >= columns), so a matrix may be some columns of a
 * wider record. dtype is the element type of every matrix and vector of a
 * call unless its comment says otherwise. Sums, softmax statistics and
 * activations are evaluated in 32 bits (matrix products of MSPLAT_DTYPE_F32
 * keep all 24 bits of both factors) and rounded once into the output's type. The
 * tensor cores truncate where they add: sums of products of one sign are off by at
 * most 4e-6 of themselves for MSPLAT_DTYPE_F32, and for the 16-bit types by 3e-5
 * (MSPLAT_DTYPE_F32 outputs, logits) or 2e-4 (the others), with up to 2^20 products.
 * Infinities and NaN act as in the formulas, except that an infinite factor of
 * MSPLAT_DTYPE_F32 may give NaN in place of an infinity beside a factor of 256 or
 * more, or below 2^-126, in size; MSPLAT_DTYPE_F32 factors below 1e-30 may lose
 * their lowest bits. Whatever lies in the other columns of a
 * wider record is neither used nor written, but 16-byte pieces of it between the
 * first and the last element of a matrix may be read.
 *
 * Calls are asynchronous on `stream`, allocate no device memory, keep nothing
 * between calls (but what msplat_ops_status says) and may be captured into a CUDA
 * graph. Sizes are at most 2^30. Working memory comes from the caller: *_workspace gives its size in bytes, the pointer must be 256-byte
 * aligned, and two calls that may run at the same time (on two streams, or in
 * two graphs) need two of them. Results do not depend on the order in which
 * blocks run. Outputs must not overlap inputs or one another unless a comment
 * allows it. Errors are returned as in msplat_backend.h (MSPLAT_OK or an
 * MSPLAT_ERR_* code, msplat_last_error()); a refused call writes nothing.
 */
#ifndef MSPLAT_OPS_H
#define MSPLAT_OPS_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types (the codes of MsplatTensorRef.dtype, continued). */
enum { MSPLAT_DTYPE_F32 = 0, MSPLAT_DTYPE_F16 = 4, MSPLAT_DTYPE_BF16 = 5 };

/* Activations: identity, max(z, 0), z Phi(z) (the exact Gaussian form),
 * z / (1 + exp(-z)), 1 / (1 + exp(-z)). */
enum {
    MSPLAT_ACT_NONE = 0,
    MSPLAT_ACT_RELU = 1,
    MSPLAT_ACT_GELU = 2,
    MSPLAT_ACT_SILU = 3,
    MSPLAT_ACT_SIGMOID = 4
};

/* z = x w^T + bias, y = act(z) + residual for x [m,k], w [n,k], bias [n] (may
 * be NULL), residual [m,n] (may be NULL) and y [m,n]; z is also written to
 * preact [m,n] when that is not NULL (msplat_linear_backward reads it, if y_dtype
 * is dtype).
 * residual, preact and y have the type y_dtype: dtype, or MSPLAT_DTYPE_F32.
 * residual may be the same memory as y (then ldr == ldy). m may be 0; n and k
 * are at least 1, and m, n, k at most 2^30. Needs no workspace. */
int msplat_linear_forward(int64_t m, int64_t n, int64_t k, const void* x, int64_t ldx, const void* w, int64_t ldw,
                          const void* bias, int32_t activation, const void* residual, int64_t ldr, void* preact,
                          int64_t ldz, void* y, int64_t ldy, int32_t dtype, int32_t y_dtype, void* stream);

/* Gradients of msplat_linear_forward from dy = dL/dy [m,n]:
 * dz = dy act'(z), dx = dz w [m,k], dw = dz^T x [n,k], dbias = column sums of
 * dz [n]; dL/dresidual is dy itself. Each of dx, dw, dbias may be NULL.
 * preact is z as a forward with y_dtype = dtype wrote it; it is not read (may be
 * NULL) for MSPLAT_ACT_NONE. x may be NULL without dw, w without dx. dx, dw and dbias are
 * overwritten, with zeros in dw and dbias when m is 0. Every matrix has the
 * type dtype; for the 16-bit types dz is rounded to dtype between the two
 * products. */
int msplat_linear_backward_workspace(int64_t m, int64_t n, int64_t k, int32_t activation, int32_t dtype,
                                     uint64_t* bytes);
int msplat_linear_backward(int64_t m, int64_t n, int64_t k, const void* x, int64_t ldx, const void* w, int64_t ldw,
                           const void* preact, int64_t ldz, int32_t activation, const void* dy, int64_t lddy,
                           void* dx, int64_t lddx, void* dw, int64_t lddw, void* dbias, int32_t dtype,
                           void* workspace, uint64_t workspace_bytes, void* stream);

/* y = residual + x * keep / (1 - p) for x, residual (may be NULL) and y
 * [rows, cols]. The mask is never stored: element e = row * cols + col draws
 * 16 bits from Philox4x32-10 (Salmon et al., SC 2011) with the key
 * (seed low, seed high) and the counter (e / 8 low, e / 8 high, c low,
 * c high), c = offset + *offset_dev (offset_dev: a device uint64, may be NULL;
 * it lets a captured graph draw another mask at every replay); draw e % 8 of a
 * block is the low half (even) or high half (odd) of its word (e % 8) / 2. The
 * element is kept when the draw is at least T = floor(65536 p + 0.5), and kept
 * elements are scaled by 65536 / (65536 - T), so p acts in steps of 2^-16.
 * Dropped elements contribute exact zeros whatever they hold. p in [0, 1];
 * p = 1 drops everything. The mask depends only on seed, c and the shape, so
 * the gradient with respect to x is the same call on dL/dy (without the
 * residual). y may be the same memory as x or residual (with the same ld). */
int msplat_dropout(int64_t rows, int64_t cols, const void* x, int64_t ldx, const void* residual, int64_t ldr,
                   void* y, int64_t ldy, float p, uint64_t seed, uint64_t offset, const uint64_t* offset_dev,
                   int32_t dtype, void* stream);

/* Softmax cross entropy of x [m,d] (one row per Gaussian or pixel) against a
 * table of label embeddings w [v,d], with its gradients, in pieces: the [m,v]
 * logits are never kept.
 *   l = logit_scale * x w^T,  row_loss[i] = log(sum_j exp(l[i,j])) - l[i,t_i]
 *   loss = weight * (sum of row_loss) / (number of labelled rows)
 * targets: int32 [m]; a row whose target lies outside [0, v) has no label: its
 * row_loss and its row of dx are 0 and it adds nothing to loss and dw, whatever
 * x holds there. Without any labelled row the loss and the gradients are 0.
 * loss (one float), row_loss (float [m]), dx [m,d] and dw [v,d] may each be
 * NULL; what is given is overwritten. The 16-bit types round the softmax
 * minus the one-hot to dtype between the products (MSPLAT_DTYPE_F16 times
 * 2^14, so that small probabilities keep their bits). m may be 0; v and d are
 * at least 1, and m, v, d at most 2^30. logit_scale and weight are
 * finite. */
int msplat_loss_cross_entropy_workspace(int64_t m, int64_t v, int64_t d, int32_t grad, int32_t dtype,
                                        uint64_t* bytes);
int msplat_loss_cross_entropy(int64_t m, int64_t v, int64_t d, const void* x, int64_t ldx, const void* w,
                              int64_t ldw, const int32_t* targets, float logit_scale, float weight, float* loss,
                              float* row_loss, void* dx, int64_t lddx, void* dw, int64_t lddw, int32_t dtype,
                              void* workspace, uint64_t workspace_bytes, void* stream);

/* Waits for `stream`, then MSPLAT_OK, or MSPLAT_ERR_CUDA when a kernel of this
 * file, on any stream of the same device, gave up waiting for its own copies or
 * products since the last call for this stream (the first call: since the library
 * was loaded). Its waits are bounded; its results are then not valid. Each
 * stream's call tells of each failure once, so none is lost to another stream's
 * call. One number per stream that has asked is kept. Not for use while a stream
 * is being captured. */
int msplat_ops_status(void* stream);

/* Launches a kernel that waits one millisecond for something that never comes and
 * gives up, as a kernel of `kernels` (0: 16-bit products, 1: other products, 2:
 * many rows against a small matrix) would: for trying how a program deals with
 * what msplat_ops_status then returns. No other result is touched. */
int msplat_ops_rehearse_timeout(int32_t kernels, void* stream);

#ifdef __cplusplus
}
#endif
#endif
