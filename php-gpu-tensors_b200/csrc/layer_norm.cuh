// Layer norm over the last axis, forwards and backwards.
//
//   m = mean(x), v = mean((x - m)^2), s = 1 / sqrt(v + eps), n = (x - m) s
//   y = n g + b
// and with a = dy g, per row and, for the parameters, over all rows
//   dx = s (a - mean(a) - n mean(a n)),  dg = sum dy n,  db = sum dy.
//
// Both directions are bound by memory: forwards reads x and writes y,
// backwards reads x and dy and writes dx, each once.  A group of TPR threads
// holds one row in registers, so the variance is taken around the mean that
// was found first (no cancellation) without a second read.  All sums are in
// float32.  The kernels come in vector widths of 16 down to 2 bytes: the widest
// one that every row start is aligned to.
//
// Backwards, thread t of a group owns the same columns of every row it meets, so
// the sums over rows stay in its registers; each block adds its groups' sums
// in shared memory and writes one partial row per parameter, and a second
// launch adds the partial rows in order (no atomics: the result does not
// depend on timing).
#pragma once

#include "ptx_sm100.cuh"
#include "rows.cuh"

namespace ptg {

struct LayerNormParams {
    const void *x, *grad, *gamma, *beta;
    void *out;                      // y, or dx
    float *mean, *rstd;             // written forwards (may be null), read backwards
    float *partial;                 // backwards: [blocks][2][cols]
    RowView xv, gv;                 // rows of x and of grad
    long long x_inner, g_inner;     // element stride of the last axis
    long long rows;
    int cols;
    float eps;
    int gamma_f32, beta_f32;        // parameters held in float32
};

// Sum over the TPR = blockDim.x threads of a row's group; `buf` is a shared
// array with a place for each warp of the block, a different array for each
// sum between two barriers.
template <int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float (*buf)[32], int tpr)
{
    const int span = tpr < 32 ? tpr : 32;
    for (int o = span / 2; o > 0; o >>= 1) {
#pragma unroll
        for (int i = 0; i < N; i++)
            v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    }
    if (tpr <= 32)
        return;
    const int lane = threadIdx.x & 31, nw = tpr >> 5, w0 = threadIdx.y * nw;
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < N; i++)
            buf[i][w0 + (threadIdx.x >> 5)] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++)
        v[i] = lane < nw ? buf[i][w0 + lane] : 0.0f;
    for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
        for (int i = 0; i < N; i++)
            v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    }
}

// VB-byte vector `c` of a row (of single elements when VB is one element,
// which also serves a strided last axis).
template <typename T, int VB>
__device__ __forceinline__ typename RawVec<VB>::type load_row_vec(const T *row, int c,
                                                                  long long inner)
{
    constexpr int E = VB / sizeof(T);
    const T *q = E == 1 ? row + c * inner : row + static_cast<long long>(c) * E;
    return __ldg(reinterpret_cast<const typename RawVec<VB>::type *>(q));
}

template <typename T, int VB, int NV>
__global__ void __launch_bounds__(512) layer_norm_kernel(const LayerNormParams p)
{
    constexpr int E = VB / sizeof(T);
    __shared__ float buf[2][1][32];
    grid_dependency_wait();
    grid_launch_dependents();
    const int tpr = blockDim.x, t = threadIdx.x;
    const int nvec = p.cols / E;
    const float inv = 1.0f / static_cast<float>(p.cols);
    const long long r = static_cast<long long>(blockIdx.x) * blockDim.y + threadIdx.y;
    const bool live = r < p.rows;
    float x[NV][E];
    float sum[1] = {0.0f};
    const T *row = static_cast<const T *>(p.x) + (live ? row_offset(p.xv, r) : 0);
#pragma unroll
    for (int v = 0; v < NV; v++) {
        const int c = v * tpr + t;
        if (live && c < nvec) {
            unpack_vec<T, VB>(load_row_vec<T, VB>(row, c, p.x_inner), x[v]);
#pragma unroll
            for (int i = 0; i < E; i++)
                sum[0] += x[v][i];
        }
    }
    group_sum(sum, buf[0], tpr);
    const float mean = sum[0] * inv;
    float var[1] = {0.0f};
#pragma unroll
    for (int v = 0; v < NV; v++) {
        if (live && v * tpr + t < nvec) {
#pragma unroll
            for (int i = 0; i < E; i++) {
                x[v][i] -= mean;
                var[0] = fmaf(x[v][i], x[v][i], var[0]);
            }
        }
    }
    group_sum(var, buf[1], tpr);
    if (!live)
        return;
    const float rstd = 1.0f / sqrtf(var[0] * inv + p.eps);
    if (t == 0 && p.mean) {
        p.mean[r] = mean;
        p.rstd[r] = rstd;
    }
    T *out = static_cast<T *>(p.out) + r * p.cols;
#pragma unroll
    for (int v = 0; v < NV; v++) {
        const int c = v * tpr + t;
        if (c < nvec) {
            float g[E], b[E];
#pragma unroll
            for (int i = 0; i < E; i++) {
                g[i] = 1.0f;
                b[i] = 0.0f;
            }
            if (p.gamma)
                load_params<T, E>(p.gamma, p.gamma_f32, static_cast<long long>(c) * E, g);
            if (p.beta)
                load_params<T, E>(p.beta, p.beta_f32, static_cast<long long>(c) * E, b);
#pragma unroll
            for (int i = 0; i < E; i++)
                x[v][i] = fmaf(x[v][i] * rstd, g[i], b[i]);
            *reinterpret_cast<typename RawVec<VB>::type *>(out + static_cast<long long>(c) * E) =
                pack_vec<T, VB>(x[v]);
        }
    }
}

// Rows too long for the registers of 512 threads: one block a row, which it
// reads three times (the second and third mostly from L2).
template <typename T>
__global__ void __launch_bounds__(512) layer_norm_long_kernel(const LayerNormParams p)
{
    __shared__ float buf[2][1][32];
    grid_dependency_wait();
    grid_launch_dependents();
    const float inv = 1.0f / static_cast<float>(p.cols);
    for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T *row = static_cast<const T *>(p.x) + row_offset(p.xv, r);
        float sum[1] = {0.0f}, var[1] = {0.0f};
        for (int c = threadIdx.x; c < p.cols; c += blockDim.x)
            sum[0] += to_float(row[c * p.x_inner]);
        group_sum(sum, buf[0], blockDim.x);
        const float mean = sum[0] * inv;
        for (int c = threadIdx.x; c < p.cols; c += blockDim.x) {
            const float d = to_float(row[c * p.x_inner]) - mean;
            var[0] = fmaf(d, d, var[0]);
        }
        group_sum(var, buf[1], blockDim.x);
        const float rstd = 1.0f / sqrtf(var[0] * inv + p.eps);
        if (threadIdx.x == 0 && p.mean) {
            p.mean[r] = mean;
            p.rstd[r] = rstd;
        }
        T *out = static_cast<T *>(p.out) + r * p.cols;
        for (int c = threadIdx.x; c < p.cols; c += blockDim.x) {
            float g[1] = {1.0f}, b[1] = {0.0f};
            if (p.gamma)
                load_params<T, 1>(p.gamma, p.gamma_f32, c, g);
            if (p.beta)
                load_params<T, 1>(p.beta, p.beta_f32, c, b);
            out[c] = from_float<T>(fmaf((to_float(row[c * p.x_inner]) - mean) * rstd, g[0], b[0]));
        }
    }
}

// Backwards: blocks walk the rows with a stride of the grid; the next row's
// loads are issued before the current row's sums are joined.
template <typename T, int VB, int NV>
__global__ void __launch_bounds__(512) layer_norm_backward_kernel(const LayerNormParams p)
{
    constexpr int E = VB / sizeof(T);
    using Raw = typename RawVec<VB>::type;
    __shared__ float buf[2][2][32];
    extern __shared__ float sums[];      // [2][cols] when a block has several groups
    grid_dependency_wait();
    grid_launch_dependents();
    const int tpr = blockDim.x, t = threadIdx.x;
    const int nvec = p.cols / E;
    const float inv = 1.0f / static_cast<float>(p.cols);
    float dg[NV][E], db[NV][E], gam[NV][E];
#pragma unroll
    for (int v = 0; v < NV; v++) {
#pragma unroll
        for (int i = 0; i < E; i++) {
            dg[v][i] = db[v][i] = 0.0f;
            gam[v][i] = 1.0f;
        }
        const int c = v * tpr + t;
        if (p.gamma && c < nvec)
            load_params<T, E>(p.gamma, p.gamma_f32, static_cast<long long>(c) * E, gam[v]);
    }
    const long long step = static_cast<long long>(gridDim.x) * blockDim.y;
    const long long first = static_cast<long long>(blockIdx.x) * blockDim.y;
    Raw rx[NV], rg[NV];
    float mean = 0.0f, rstd = 0.0f;
    auto fetch = [&](long long r) {
        if (r >= p.rows)
            return;
        const T *xr = static_cast<const T *>(p.x) + row_offset(p.xv, r);
        const T *gr = static_cast<const T *>(p.grad) + row_offset(p.gv, r);
#pragma unroll
        for (int v = 0; v < NV; v++) {
            const int c = v * tpr + t;
            if (c < nvec) {
                rx[v] = load_row_vec<T, VB>(xr, c, p.x_inner);
                rg[v] = load_row_vec<T, VB>(gr, c, p.g_inner);
            }
        }
        mean = __ldg(p.mean + r);
        rstd = __ldg(p.rstd + r);
    };
    fetch(first + threadIdx.y);
    int parity = 0;
    // every group of the block makes the same number of steps
    for (long long base = first; base < p.rows; base += step, parity ^= 1) {
        const long long r = base + threadIdx.y;
        const bool live = r < p.rows;
        float n[NV][E], a[NV][E];
        float s[2] = {0.0f, 0.0f};
        const float rs = rstd;
#pragma unroll
        for (int v = 0; v < NV; v++) {
            if (live && v * tpr + t < nvec) {
                unpack_vec<T, VB>(rx[v], n[v]);
                unpack_vec<T, VB>(rg[v], a[v]);
#pragma unroll
                for (int i = 0; i < E; i++) {
                    n[v][i] = (n[v][i] - mean) * rs;
                    dg[v][i] = fmaf(a[v][i], n[v][i], dg[v][i]);
                    db[v][i] += a[v][i];
                    a[v][i] *= gam[v][i];
                    s[0] += a[v][i];
                    s[1] = fmaf(a[v][i], n[v][i], s[1]);
                }
            }
        }
        fetch(r + step);
        group_sum(s, buf[parity], tpr);
        if (live) {
            const float ma = s[0] * inv, mn = s[1] * inv;
            T *out = static_cast<T *>(p.out) + r * p.cols;
#pragma unroll
            for (int v = 0; v < NV; v++) {
                const int c = v * tpr + t;
                if (c < nvec) {
#pragma unroll
                    for (int i = 0; i < E; i++)
                        a[v][i] = rs * (a[v][i] - ma - n[v][i] * mn);
                    *reinterpret_cast<Raw *>(out + static_cast<long long>(c) * E) =
                        pack_vec<T, VB>(a[v]);
                }
            }
        }
    }
    if (!p.partial)
        return;
    float *part = p.partial + static_cast<long long>(blockIdx.x) * 2 * p.cols;
    float *dst = blockDim.y > 1 ? sums : part;
    for (int y = 0; y < static_cast<int>(blockDim.y); y++) {
        if (static_cast<int>(threadIdx.y) == y) {
#pragma unroll
            for (int v = 0; v < NV; v++) {
                const int c = (v * tpr + t) * E;
                if (v * tpr + t < nvec) {
#pragma unroll
                    for (int i = 0; i < E; i++) {
                        dst[c + i] = y == 0 ? dg[v][i] : dst[c + i] + dg[v][i];
                        dst[p.cols + c + i] =
                            y == 0 ? db[v][i] : dst[p.cols + c + i] + db[v][i];
                    }
                }
            }
        }
        if (blockDim.y > 1)
            __syncthreads();
    }
    if (blockDim.y > 1) {
        const int threads = blockDim.x * blockDim.y;
        for (int c = threadIdx.y * tpr + t; c < 2 * p.cols; c += threads)
            part[c] = sums[c];
    }
}

// Backwards for rows too long for the registers: dx, one block a row ...
template <typename T>
__global__ void __launch_bounds__(512) layer_norm_backward_long_kernel(const LayerNormParams p)
{
    __shared__ float buf[2][2][32];
    grid_dependency_wait();
    grid_launch_dependents();
    const float inv = 1.0f / static_cast<float>(p.cols);
    int parity = 0;
    for (long long r = blockIdx.x; r < p.rows; r += gridDim.x, parity ^= 1) {
        const T *xr = static_cast<const T *>(p.x) + row_offset(p.xv, r);
        const T *gr = static_cast<const T *>(p.grad) + row_offset(p.gv, r);
        const float mean = p.mean[r], rstd = p.rstd[r];
        float s[2] = {0.0f, 0.0f};
        for (int c = threadIdx.x; c < p.cols; c += blockDim.x) {
            float g[1] = {1.0f};
            if (p.gamma)
                load_params<T, 1>(p.gamma, p.gamma_f32, c, g);
            const float a = to_float(gr[c * p.g_inner]) * g[0];
            s[0] += a;
            s[1] = fmaf(a, (to_float(xr[c * p.x_inner]) - mean) * rstd, s[1]);
        }
        group_sum(s, buf[parity], blockDim.x);
        const float ma = s[0] * inv, mn = s[1] * inv;
        T *out = static_cast<T *>(p.out) + r * p.cols;
        for (int c = threadIdx.x; c < p.cols; c += blockDim.x) {
            float g[1] = {1.0f};
            if (p.gamma)
                load_params<T, 1>(p.gamma, p.gamma_f32, c, g);
            const float a = to_float(gr[c * p.g_inner]) * g[0];
            const float n = (to_float(xr[c * p.x_inner]) - mean) * rstd;
            out[c] = from_float<T>(rstd * (a - ma - n * mn));
        }
    }
}

// ... and the parameters' sums, a block taking 256 columns of every
// gridDim.y-th row.
template <typename T>
__global__ void __launch_bounds__(256) layer_norm_param_long_kernel(const LayerNormParams p)
{
    grid_dependency_wait();
    grid_launch_dependents();
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= p.cols)
        return;
    float dg = 0.0f, db = 0.0f;
    for (long long r = blockIdx.y; r < p.rows; r += gridDim.y) {
        const T *xr = static_cast<const T *>(p.x) + row_offset(p.xv, r);
        const T *gr = static_cast<const T *>(p.grad) + row_offset(p.gv, r);
        const float g = to_float(gr[c * p.g_inner]);
        dg = fmaf(g, (to_float(xr[c * p.x_inner]) - p.mean[r]) * p.rstd[r], dg);
        db += g;
    }
    float *part = p.partial + static_cast<long long>(blockIdx.y) * 2 * p.cols;
    part[c] = dg;
    part[p.cols + c] = db;
}

// out[s][c] = sum over n partial rows of partial[k][s * cols + c], in the
// order of k within each of 32 interleaved sums.  blockIdx.y = s; a null out
// is skipped.
__global__ void __launch_bounds__(1024) sum_partials_kernel(const float *partial, int n,
                                                            long long width, int cols, float *out0,
                                                            float *out1)
{
    __shared__ float acc[32][33];
    grid_dependency_wait();
    grid_launch_dependents();
    float *out = blockIdx.y == 0 ? out0 : out1;
    if (!out)
        return;
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + tx;
    float sum = 0.0f;
    if (c < cols) {
        const float *q = partial + static_cast<long long>(blockIdx.y) * cols + c;
#pragma unroll 4
        for (int k = ty; k < n; k += 32)
            sum += q[k * width];
    }
    acc[ty][tx] = sum;
    __syncthreads();
    float total = acc[tx][ty];           // column ty of the block, partial sum tx
    for (int o = 16; o > 0; o >>= 1)
        total += __shfl_xor_sync(0xffffffffu, total, o);
    const int oc = blockIdx.x * 32 + ty;
    if (tx == 0 && oc < cols)
        out[oc] = total;
}

} // namespace ptg
