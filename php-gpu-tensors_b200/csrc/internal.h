// Declarations shared by the library's translation units (not exported).
#pragma once

#include <cuda_runtime_api.h>
#include <cstddef>

// Records a status code for cuda_blas_info().last_blas_status (this thread).
void ptg_set_last_status(int code);

namespace ptg {

// Destinations of the fused N-split epilogue: this rank's column block is
// written into every rank's row-major [M, ldc] result at column col_off.
struct F64PeerOut {
    double *dst[8];
    int ndst;
    int rot;              // this rank: destination (rot + i) % ndst is stored i-th
    long long ldc;
    long long col_off;
    int exchange;         // GEMM_MGPU_EXCHANGE_*: store, overlap, or by rank count
    unsigned long long *slots;   // overlap: per-SM hand-off slots (device memory, zeroed)
    int nslots;
};

} // namespace ptg

// The float64 N-split block product whose epilogue writes into every rank's
// result: A is [M, K], B the [K, nb] block, both 2-D strided views; needs nb
// even and 16-byte aligned destinations.
cudaError_t ptg_launch_f64_peer(const double *a, size_t a_s0, size_t a_s1, const double *b,
                                size_t b_s0, size_t b_s1, int M, int nb, int K,
                                const ptg::F64PeerOut &po, cudaStream_t stream);

// float32 C = the sum over C's reduced batch axes of A . B: an axis where the
// broadcast batch shape of A and B has extent > 1 and C has extent 1 (or no
// axis) is summed inside the product kernel (the k loop runs over it), so the
// un-broadcast step of a gradient needs no scratch tensor and no second
// kernel.  Operand dtypes are dtype_t values: float32, float16, bfloat16 (not
// float16 with bfloat16).  Returns 1 / 0 like the launchers.
int ptg_reduced_matmul(const void *a, int a_dtype, const void *b, int b_dtype, float *c,
                       int *shape_a, size_t *stride_a, int nd_a, int *shape_b, size_t *stride_b,
                       int nd_b, int *shape_c, size_t *stride_c, int nd_c, cudaStream_t stream);

// ------------------------------------------------------------ feed-forward
// Device facts and launch bookkeeping of csrc/gemm_sm100.cu for the other
// translation units.  ptg_device returns false (and sets the status) without
// an sm_100 device.
struct PtgDevice {
    int sms;
    int *status;      // device status word
    void *encode;     // cuTensorMapEncodeTiled
};
bool ptg_device(PtgDevice *out);
int ptg_precision();  // CUDA_MATMUL_PRECISION_* of this thread
int ptg_path();       // gemm_sm100_set_path of this thread
// Names the thread's last kernel and clears its status; a product also counts
// as a matmul call of `dtype`'s family.
void ptg_record_launch(const char *kernel, bool product, int dtype, int grid, int block,
                       int cluster);

// Sets pt_last_error() of this thread and returns `code`; ptg_ok() clears it.
int ptg_fail(int code, const char *message);
int ptg_ok();

namespace ptg {

// The rows of a tensor: its leading axes, merged where their strides compose.
constexpr int kRowViewAxes = 4;
struct RowView {
    int n;                              // merged axes, outermost first (at least 1)
    int ext[kRowViewAxes];
    long long stride[kRowViewAxes];     // in elements
};

} // namespace ptg

// Layer norm launches (csrc/layer_norm.cu); arguments are validated by the
// caller (host/feed_forward.cpp).  dtype is a dtype_t.  Both return a
// cudaError_t.
struct PtgLayerNorm {
    int dtype;
    const void *x, *grad, *gamma, *beta;
    int gamma_f32, beta_f32;
    ptg::RowView xv, gv;
    long long x_inner, g_inner, rows;
    int cols;
    float eps;
    void *out;
    float *mean, *rstd;
    float *dgamma, *dbeta;              // backwards: either may be null
    float *partial;                     // backwards: workspace
};
cudaError_t ptg_layer_norm(const PtgLayerNorm &a, cudaStream_t stream);
cudaError_t ptg_layer_norm_backward(const PtgLayerNorm &a, cudaStream_t stream);
size_t ptg_layer_norm_partial_bytes(long long rows, int cols);

// Linear layers (csrc/linear.cu): rows in groups, each with its own weight.
// Arguments are validated by the caller (host/feed_forward.cpp).
struct PtgLinear {
    int dtype;                          // dtype_t of x, w, y, grad, dx and pre
    int groups, rows, inner, cols;      // w is [groups, inner, cols]
    const int *ends;                    // device, or null for one group of all rows
    const void *x;
    ptg::RowView xv;
    long long x_inner;
    const void *w;
    long long w_group, w_inner, w_cols; // element strides
    int activation;
    // forwards
    const void *bias;                   // [groups, cols]
    int bias_f32;
    const void *residual;
    ptg::RowView rv;
    long long r_inner;
    void *y;
    void *pre;                          // written forwards (may be null), read backwards
    // backwards
    const void *grad;
    ptg::RowView gv;
    long long g_inner;
    ptg::RowView pv;                    // rows of pre
    long long p_inner;
    void *dx, *dw;
    int dw_dtype;
    float *dbias;
    void *workspace;
    size_t workspace_bytes;
};
// Both return a cudaError_t, or cudaErrorMemoryAllocation with *need set and
// nothing enqueued when the workspace is too small.
cudaError_t ptg_linear(const PtgLinear &a, size_t *need, cudaStream_t stream);
cudaError_t ptg_linear_backward(const PtgLinear &a, size_t *need, cudaStream_t stream);
