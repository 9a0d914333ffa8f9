// Feed-forward layers at tensor level (include/pt_feed_forward.h): argument
// checks and the row views of strided tensors, above the launches of
// csrc/layer_norm.cu and csrc/linear.cu.
#include "pt_feed_forward.h"

#include "internal.h"

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>

#define PT_API extern "C" __attribute__((visibility("default")))

namespace {

int invalid(const char *message) { return ptg_fail(PT_INVALID_ARGUMENT, message); }

int submitted(cudaError_t err, const char *what)
{
    if (err == cudaSuccess)
        return ptg_ok();
    char text[160];
    std::snprintf(text, sizeof(text), "%s submission failed (CUDA error %d)", what,
                  static_cast<int>(err));
    return ptg_fail(PT_RUNTIME, text);
}

// Extents that the kernels walk with 32-bit indexes, which step up to a tile past
// the end before they are compared with it.
constexpr int kMaxExtent = 2147483647 - 1024;

bool float_type(int dtype)
{
    return dtype == DTYPE_FLOAT32 || dtype == DTYPE_FLOAT16 || dtype == DTYPE_BFLOAT16;
}

bool valid(const pt_tensor *t)
{
    if (!t || t->ndims < 1 || t->ndims > MAX_DIMS)
        return false;
    for (int d = 0; d < t->ndims; d++)
        if (t->shape[d] < 0)
            return false;
    return true;
}

int last(const pt_tensor *t) { return t->shape[t->ndims - 1]; }

// Product of the leading extents.
long long row_count(const pt_tensor *t)
{
    long long n = 1;
    for (int d = 0; d < t->ndims - 1; d++)
        n *= t->shape[d];
    return n;
}

bool same_shape(const pt_tensor *a, const pt_tensor *b)
{
    if (a->ndims != b->ndims)
        return false;
    for (int d = 0; d < a->ndims; d++)
        if (a->shape[d] != b->shape[d])
            return false;
    return true;
}

bool contiguous(const pt_tensor *t)
{
    size_t step = 1;
    for (int d = t->ndims - 1; d >= 0; d--) {
        if (t->shape[d] != 1 && t->strides[d] != step)
            return false;
        step *= static_cast<size_t>(t->shape[d]);
    }
    return true;
}

// Merges the leading axes.  Returns false when more than kRowViewAxes remain.
bool row_view(const pt_tensor *t, ptg::RowView *v)
{
    std::memset(v, 0, sizeof(*v));
    int ext[MAX_DIMS];
    long long stride[MAX_DIMS];
    int n = 0;
    for (int d = 0; d < t->ndims - 1; d++) {
        const int e = t->shape[d];
        const long long s = static_cast<long long>(t->strides[d]);
        if (e == 1)
            continue;
        if (n > 0 && stride[n - 1] == s * e &&
            static_cast<long long>(ext[n - 1]) * e < (1ll << 31)) {
            ext[n - 1] *= e;
            stride[n - 1] = s;
        } else {
            ext[n] = e;
            stride[n++] = s;
        }
    }
    if (n == 0) {
        ext[0] = 1;
        stride[0] = 0;
        n = 1;
    }
    if (n > ptg::kRowViewAxes)
        return false;
    v->n = n;
    for (int d = 0; d < n; d++) {
        v->ext[d] = ext[d];
        v->stride[d] = stride[d];
    }
    return true;
}

// A [cols] vector of x's type or float32.
bool parameter(const pt_tensor *p, const pt_tensor *x, int cols)
{
    return !p || (p->ndims == 1 && p->shape[0] == cols && (cols <= 1 || p->strides[0] == 1) &&
                  (p->dtype == x->dtype || p->dtype == DTYPE_FLOAT32));
}

const void *data(const pt_tensor *t) { return t ? t->data : nullptr; }

} // namespace

// ------------------------------------------------------------ layer norm
PT_API int pt_layer_norm(const pt_tensor *x, const pt_tensor *gamma, const pt_tensor *beta,
                         float eps, const pt_tensor *y, float *mean, float *rstd,
                         cudaStream_t stream)
{
    if (!valid(x) || !valid(y) || !float_type(x->dtype) || y->dtype != x->dtype)
        return invalid("layer norm requires a float32, float16 or bfloat16 tensor");
    const int cols = last(x);
    if (cols < 1)
        return invalid("layer norm requires at least one column");
    if (cols > kMaxExtent)
        return invalid("layer norm takes fewer than 2^31 - 1024 columns");
    if (!parameter(gamma, x, cols) || !parameter(beta, x, cols))
        return invalid("layer norm gamma and beta must be [cols] vectors of the tensor's type or "
                       "float32");
    if (!same_shape(x, y) || !contiguous(y))
        return invalid("layer norm writes a contiguous result of the tensor's shape");
    if (!(eps >= 0.0f) || !std::isfinite(eps))
        return invalid("layer norm eps must be finite and not negative");
    if ((mean == nullptr) != (rstd == nullptr))
        return invalid("layer norm writes both statistics or neither");
    PtgLayerNorm a;
    std::memset(&a, 0, sizeof(a));
    if (!row_view(x, &a.xv))
        return invalid("layer norm cannot merge the tensor's leading axes");
    a.rows = row_count(x);
    if (a.rows == 0)
        return ptg_ok();
    if (!x->data || !y->data || (gamma && !gamma->data) || (beta && !beta->data))
        return invalid("layer norm got a null pointer");
    a.dtype = x->dtype;
    a.x = x->data;
    a.gamma = data(gamma);
    a.beta = data(beta);
    a.gamma_f32 = gamma && gamma->dtype == DTYPE_FLOAT32;
    a.beta_f32 = beta && beta->dtype == DTYPE_FLOAT32;
    a.x_inner = cols == 1 ? 1 : static_cast<long long>(x->strides[x->ndims - 1]);
    a.cols = cols;
    a.eps = eps;
    a.out = y->data;
    a.mean = mean;
    a.rstd = rstd;
    return submitted(ptg_layer_norm(a, stream), "Layer norm");
}

PT_API size_t pt_layer_norm_backward_workspace(long long rows, int cols)
{
    return rows > 0 && cols > 0 ? ptg_layer_norm_partial_bytes(rows, cols) : 0;
}

PT_API int pt_layer_norm_backward(const pt_tensor *grad, const pt_tensor *x,
                                  const pt_tensor *gamma, const float *mean, const float *rstd,
                                  const pt_tensor *dx, float *dgamma, float *dbeta,
                                  void *workspace, size_t *workspace_bytes, cudaStream_t stream)
{
    if (!valid(grad) || !valid(x) || !valid(dx) || !float_type(x->dtype) ||
        grad->dtype != x->dtype || dx->dtype != x->dtype)
        return invalid("layer norm requires a float32, float16 or bfloat16 tensor");
    const int cols = last(x);
    if (cols < 1)
        return invalid("layer norm requires at least one column");
    if (cols > kMaxExtent)
        return invalid("layer norm takes fewer than 2^31 - 1024 columns");
    if (!parameter(gamma, x, cols))
        return invalid("layer norm gamma and beta must be [cols] vectors of the tensor's type or "
                       "float32");
    if (!same_shape(x, grad))
        return invalid("layer norm needs an upstream gradient of the tensor's shape");
    if (!same_shape(x, dx) || !contiguous(dx))
        return invalid("layer norm writes a contiguous result of the tensor's shape");
    PtgLayerNorm a;
    std::memset(&a, 0, sizeof(a));
    if (!row_view(x, &a.xv) || !row_view(grad, &a.gv))
        return invalid("layer norm cannot merge the tensor's leading axes");
    a.rows = row_count(x);
    if (a.rows == 0) {
        cudaError_t err = cudaSuccess;
        if (dgamma)
            err = cudaMemsetAsync(dgamma, 0, static_cast<size_t>(cols) * 4, stream);
        if (dbeta && err == cudaSuccess)
            err = cudaMemsetAsync(dbeta, 0, static_cast<size_t>(cols) * 4, stream);
        return submitted(err, "Layer norm gradient");
    }
    if (!x->data || !grad->data || !dx->data || !mean || !rstd || (gamma && !gamma->data))
        return invalid("layer norm got a null pointer");
    if (dgamma || dbeta) {
        const size_t need = ptg_layer_norm_partial_bytes(a.rows, cols);
        if (!workspace_bytes || !workspace || *workspace_bytes < need) {
            if (workspace_bytes)
                *workspace_bytes = need;
            return ptg_fail(PT_WORKSPACE, "layer norm gradient needs a larger workspace");
        }
        if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
            return invalid("the workspace must be aligned to 16 bytes");
    }
    a.dtype = x->dtype;
    a.x = x->data;
    a.grad = grad->data;
    a.gamma = data(gamma);
    a.gamma_f32 = gamma && gamma->dtype == DTYPE_FLOAT32;
    a.x_inner = cols == 1 ? 1 : static_cast<long long>(x->strides[x->ndims - 1]);
    a.g_inner = cols == 1 ? 1 : static_cast<long long>(grad->strides[grad->ndims - 1]);
    a.cols = cols;
    a.out = dx->data;
    a.mean = const_cast<float *>(mean);
    a.rstd = const_cast<float *>(rstd);
    a.dgamma = dgamma;
    a.dbeta = dbeta;
    a.partial = static_cast<float *>(workspace);
    return submitted(ptg_layer_norm_backward(a, stream), "Layer norm gradient");
}

// ------------------------------------------------------------ linear layers
namespace {

// The layer's shapes and operands that both directions share; PT_OK or a
// refusal.  `out` has the result's (or the gradient's) shape.
int layer(const pt_tensor *x, const pt_tensor *w, const int *ends, int activation,
          const pt_tensor *out, PtgLinear *a)
{
    std::memset(a, 0, sizeof(*a));
    if (!valid(x) || !valid(w) || !valid(out) || !float_type(x->dtype) ||
        w->dtype != x->dtype || out->dtype != x->dtype)
        return invalid("linear layers require matching float32, float16 or bfloat16 tensors");
    if (w->ndims != (ends ? 3 : 2))
        return invalid(ends ? "a grouped linear layer needs a [groups, inner, cols] weight and ends"
                            : "a linear layer needs a [inner, cols] weight");
    if (x->ndims < 2 || (ends && x->ndims != 2) || out->ndims != x->ndims)
        return invalid("linear layers require rows of the inner size");
    const int d = w->ndims;
    a->groups = ends ? w->shape[0] : 1;
    a->inner = w->shape[d - 2];
    a->cols = w->shape[d - 1];
    if (last(x) != a->inner || last(out) != a->cols)
        return invalid("linear layer shapes do not match");
    for (int i = 0; i < x->ndims - 1; i++)
        if (x->shape[i] != out->shape[i])
            return invalid("linear layer shapes do not match");
    if (activation < CUDA_MATMUL_EPILOGUE_NONE || activation > CUDA_MATMUL_EPILOGUE_SILU)
        return invalid("linear layer activation is unknown");
    const long long rows = row_count(x);
    if (a->groups < 1 || a->groups > PT_MAX_GROUPS)
        return invalid("a grouped linear layer takes 1 to 2048 groups");
    if (rows > kMaxExtent || a->inner > kMaxExtent || a->cols > kMaxExtent)
        return invalid("linear layers take fewer than 2^31 - 1024 rows, inner elements and columns");
    if (!row_view(x, &a->xv))
        return invalid("linear layer cannot merge the tensor's leading axes");
    a->dtype = x->dtype;
    a->rows = static_cast<int>(rows);
    a->ends = ends;
    a->x = x->data;
    a->x_inner = static_cast<long long>(x->strides[x->ndims - 1]);
    a->w = w->data;
    a->w_group = ends ? static_cast<long long>(w->strides[0]) : 0;
    a->w_inner = static_cast<long long>(w->strides[d - 2]);
    a->w_cols = static_cast<long long>(w->strides[d - 1]);
    a->activation = activation;
    return PT_OK;
}

// Runs `call` on the caller's workspace.
template <typename F>
int with_workspace(PtgLinear *a, void *workspace, size_t *workspace_bytes, const char *what, F call)
{
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
        return invalid("the workspace must be aligned to 16 bytes");
    a->workspace = workspace;
    a->workspace_bytes = workspace && workspace_bytes ? *workspace_bytes : 0;
    size_t need = 0;
    const cudaError_t err = call(*a, &need);
    if (err == cudaErrorMemoryAllocation && need > a->workspace_bytes) {
        if (workspace_bytes)
            *workspace_bytes = need;
        return ptg_fail(PT_WORKSPACE, "linear layer needs a larger workspace");
    }
    return submitted(err, what);
}

} // namespace

PT_API int pt_linear(const pt_tensor *x, const pt_tensor *w, const int *ends,
                     const pt_tensor *bias, int activation, const pt_tensor *residual,
                     const pt_tensor *y, const pt_tensor *pre, void *workspace,
                     size_t *workspace_bytes, cudaStream_t stream)
{
    PtgLinear a;
    if (const int refused = layer(x, w, ends, activation, y, &a))
        return refused;
    if (!contiguous(y) || (pre && (!valid(pre) || pre->dtype != x->dtype || !same_shape(pre, y) ||
                                   !contiguous(pre))))
        return invalid("linear layers write contiguous results");
    if (bias) {
        const bool shaped = valid(bias) && bias->ndims == w->ndims - 1 &&
                            (!ends || bias->shape[0] == a.groups) && last(bias) == a.cols;
        if (!shaped || !contiguous(bias) ||
            (bias->dtype != x->dtype && bias->dtype != DTYPE_FLOAT32))
            return invalid("linear layer bias must be a contiguous [cols] or [groups, cols] tensor "
                           "of the operands' type or float32");
    }
    if (residual && (!valid(residual) || residual->dtype != x->dtype || !same_shape(residual, y)))
        return invalid("linear layer residual must have the result's shape and type");
    if (residual && !row_view(residual, &a.rv))
        return invalid("linear layer cannot merge the tensor's leading axes");
    if (a.rows == 0 || a.cols == 0)
        return ptg_ok();
    if (!y->data || (a.inner > 0 && (!x->data || !w->data)) || (bias && !bias->data) ||
        (residual && !residual->data) || (pre && !pre->data))
        return invalid("linear layer got a null pointer");
    a.bias = data(bias);
    a.bias_f32 = bias && bias->dtype == DTYPE_FLOAT32;
    a.residual = data(residual);
    a.r_inner = residual ? static_cast<long long>(residual->strides[residual->ndims - 1]) : 0;
    a.y = y->data;
    a.pre = pre ? pre->data : nullptr;
    return with_workspace(&a, workspace, workspace_bytes, "Linear layer",
                          [&](const PtgLinear &l, size_t *need) {
                              return ptg_linear(l, need, stream);
                          });
}

PT_API int pt_linear_backward(const pt_tensor *grad, const pt_tensor *x, const pt_tensor *w,
                              const int *ends, const pt_tensor *pre, int activation,
                              const pt_tensor *dx, const pt_tensor *dw, float *dbias,
                              void *workspace, size_t *workspace_bytes, cudaStream_t stream)
{
    PtgLinear a;
    if (const int refused = layer(x, w, ends, activation, grad, &a))
        return refused;
    if (!row_view(grad, &a.gv))
        return invalid("linear layer cannot merge the tensor's leading axes");
    if (activation == CUDA_MATMUL_EPILOGUE_NONE)
        pre = nullptr;
    else if (!valid(pre) || pre->dtype != x->dtype || !same_shape(pre, grad) ||
             !row_view(pre, &a.pv))
        return invalid("linear layer gradient needs the pre-activation, of the result's shape and "
                       "type");
    if (dx && (!valid(dx) || dx->dtype != x->dtype || !same_shape(dx, x) || !contiguous(dx)))
        return invalid("linear layer dx must be contiguous, of the input's shape and type");
    if (dw && (!valid(dw) || (dw->dtype != x->dtype && dw->dtype != DTYPE_FLOAT32) ||
               !same_shape(dw, w) || !contiguous(dw)))
        return invalid("linear layer dw must be contiguous, of the weight's shape and its type or "
                       "float32");
    const size_t weights = static_cast<size_t>(a.groups) * a.inner * a.cols;
    if (a.inner == 0 || a.cols == 0 || a.rows == 0) {
        // sums over nothing
        cudaError_t err = cudaSuccess;
        if (dx && dx->data && a.rows > 0 && a.inner > 0)
            err = cudaMemsetAsync(dx->data, 0, static_cast<size_t>(a.rows) * a.inner *
                                  (a.dtype == DTYPE_FLOAT32 ? 4 : 2), stream);
        if (err == cudaSuccess && dw && dw->data && weights > 0)
            err = cudaMemsetAsync(dw->data, 0, weights * (dw->dtype == DTYPE_FLOAT32 ? 4 : 2),
                                  stream);
        if (err != cudaSuccess || a.rows == 0 || a.cols == 0) {
            if (err == cudaSuccess && dbias && a.cols > 0)
                err = cudaMemsetAsync(dbias, 0, static_cast<size_t>(a.groups) * a.cols * 4, stream);
            return submitted(err, "Linear layer gradient");
        }
        dx = dw = nullptr;
    }
    if (!grad->data || ((dx || dw) && (!x->data || !w->data)) || (pre && !pre->data) ||
        (dx && !dx->data) || (dw && !dw->data))
        return invalid("linear layer got a null pointer");
    a.grad = grad->data;
    a.g_inner = static_cast<long long>(grad->strides[grad->ndims - 1]);
    a.pre = pre ? pre->data : nullptr;
    a.p_inner = pre ? static_cast<long long>(pre->strides[pre->ndims - 1]) : 0;
    a.dx = dx ? dx->data : nullptr;
    a.dw = dw ? dw->data : nullptr;
    a.dw_dtype = dw ? dw->dtype : 0;
    a.dbias = dbias;
    if (!a.dx && !a.dw && !a.dbias)
        return ptg_ok();
    return with_workspace(&a, workspace, workspace_bytes, "Linear layer gradient",
                          [&](const PtgLinear &l, size_t *need) {
                              return ptg_linear_backward(l, need, stream);
                          });
}
