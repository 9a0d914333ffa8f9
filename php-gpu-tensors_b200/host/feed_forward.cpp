// Feed-forward layers at tensor level (include/pt_feed_forward.h): argument
// checks, the row views of strided tensors, and workspace layout, above the
// launches of csrc/layer_norm.cu.
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
