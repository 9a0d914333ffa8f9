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
 * mode (cuda_blas_set_precision).
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

#ifdef __cplusplus
}
#endif

#endif /* PT_FEED_FORWARD_H */
