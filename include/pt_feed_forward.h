/*
 * pt_feed_forward.h -- the layers around the products of a feed-forward
 * block: layer norm, the linear layer with bias, activation and residual in
 * its epilogue, and the same layer grouped by expert; forwards and backwards.
 * No counterpart in the reference, whose tensors have the product alone.
 *
 * Conventions are those of pt_tensor.h and gemm_sm100.h: tensors describe
 * device memory with strides in elements, results are preallocated,
 * contiguous and row-major and overlap no input, work is enqueued on `stream`
 * without allocating, synchronising or reading device memory on the host, and
 * every function returns PT_OK or a PT_* code with pt_last_error() set.
 * Operands are float32, float16 or bfloat16, all of one type unless said
 * otherwise; sums, statistics and activations are computed in float32 and a
 * result is rounded once.  float32 products follow the thread's precision
 * mode (cuda_blas_set_precision).  Columns, inner elements and the linear layers'
 * rows number fewer than 2^31 - 1024 each; offsets are 64-bit.
 */
#ifndef PT_FEED_FORWARD_H
#define PT_FEED_FORWARD_H

#include "pt_tensor.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The workspace passed is smaller than the call needs: nothing was enqueued,
 * *workspace_bytes holds the need. */
#define PT_WORKSPACE 3

/* Layer norm over the last axis: y = (x - mean) / sqrt(var + eps) * gamma +
 * beta, var the mean square distance from the mean.  x has rank 1 to
 * MAX_DIMS; its leading axes may have any strides that merge into at most
 * four.  gamma and beta are contiguous [cols] vectors of x's type or float32,
 * or NULL (1 and 0).  mean and rstd, both or neither NULL, receive one
 * float32 per row for the backward pass. */
int pt_layer_norm(const pt_tensor *x, const pt_tensor *gamma, const pt_tensor *beta, float eps,
                  const pt_tensor *y, float *mean, float *rstd, cudaStream_t stream);

/* Gradients of pt_layer_norm for the upstream gradient `grad` (x's shape and
 * type): dx in x's type, and the sums over all rows dgamma and dbeta, [cols]
 * float32 as the gradients of this library's products are (either may be
 * NULL).  With one of them given the call needs
 * pt_layer_norm_backward_workspace(rows, cols) bytes. */
int pt_layer_norm_backward(const pt_tensor *grad, const pt_tensor *x, const pt_tensor *gamma,
                           const float *mean, const float *rstd, const pt_tensor *dx,
                           float *dgamma, float *dbeta, void *workspace, size_t *workspace_bytes,
                           cudaStream_t stream);
size_t pt_layer_norm_backward_workspace(long long rows, int cols);

/* Linear layer y = activation(x . w + bias) + residual.
 *
 * x is [..., K]; its leading axes are the rows.  Without `ends` w is [K, N].
 * With `ends` the layer is grouped by expert: w is [E, K, N], x is [rows, K]
 * with the rows sorted by group, and ends, E int32 on the device, holds the
 * row behind each group's last one (the running sum of the groups' row
 * counts; an empty group repeats the value before it).  Values that fall or
 * pass the row count are read as the nearest allowed one; rows behind the
 * last group belong to none and get zeros.  At most PT_MAX_GROUPS groups.
 * x, w and residual may have any strides (leading axes as for the layer
 * norm); operands that the tensor cores' loads cannot describe (no contiguous
 * axis, rows that do not start at multiples of 16 bytes) are laid out in the
 * workspace first, and so are the bfloat16 parts of float32 ones.
 *
 * bias is contiguous [N] ([E, N]) of x's type or float32; residual has y's
 * shape and x's type; activation is a CUDA_MATMUL_EPILOGUE_* value.  RELU is
 * z > 0 ? z : 0 as in the matmul's epilogue, so that NaN becomes 0 there (and its
 * slope 0); the other activations keep it.  y and, unless NULL,
 * pre = x . w + bias, which the backward pass needs for an activation, are
 * [..., N] of x's type.  Infinite float32 operands, and finite ones that round to
 * infinity in bfloat16 (from 3.396e38 on), can turn to NaN as in the strict mode of
 * cuda_blas_set_precision.
 *
 * *workspace_bytes holds the size of `workspace` (16-byte aligned); where it
 * is too small the call returns PT_WORKSPACE with the need in its place. */
#define PT_MAX_GROUPS 2048
int pt_linear(const pt_tensor *x, const pt_tensor *w, const int *ends, const pt_tensor *bias,
              int activation, const pt_tensor *residual, const pt_tensor *y,
              const pt_tensor *pre, void *workspace, size_t *workspace_bytes,
              cudaStream_t stream);

/* Gradients of pt_linear for the upstream gradient `grad` (y's shape, x's
 * type): with dz = grad * activation'(pre)
 *     dx = dz . w^T       [..., K], x's type
 *     dw = x^T . dz       w's shape (contiguous), x's type or float32
 *     dbias = column sums of dz, float32 [N] ([E, N])
 * each unless NULL; the residual's gradient is grad itself.  pre may be NULL
 * for CUDA_MATMUL_EPILOGUE_NONE.  For 16-bit operands dz is rounded to their
 * type before the two products, except where these run on the CUDA cores: where
 * dz has no more than 16384 elements (unless gemm_sm100_set_path chose 1 or 3), for
 * small products of operands that would have to be laid out, and where path 2
 * was chosen.  There it stays in float32, whatever type dw is wanted in.
 * dbias is summed before the rounding; without an activation grad is used as it is.
 * Rows of no group take no part, and their dx is zero; a group without rows has
 * a gradient of zero. */
int pt_linear_backward(const pt_tensor *grad, const pt_tensor *x, const pt_tensor *w,
                       const int *ends, const pt_tensor *pre, int activation,
                       const pt_tensor *dx, const pt_tensor *dw, float *dbias, void *workspace,
                       size_t *workspace_bytes, cudaStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* PT_FEED_FORWARD_H */
