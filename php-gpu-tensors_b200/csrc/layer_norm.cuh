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
//
// On B200, with the time of the bytes at the copy rate behind it: 16384 x 4096
// bfloat16 forwards 84 us (41), backwards 84 and 5 for the partial rows (62); one
// row ahead is what the registers hold, and more loads in flight have been tried
// only before the arithmetic was packed (bulk copies into shared memory, 116 us).
// 3001 x 1531 float32 forwards 14 us (5.6) and 17 alone, of which a launch takes
// about five: 4-byte loads, as its rows start at every alignment.  8192 x 1024
// float32 16 (10) and 26 (15); 4096 x 12288 bfloat16 61 (31) and, on the kernels for
// long rows with their three reads of single elements, 340 (46).
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
        v[i] = buf[i][w0 + (lane & (nw - 1))];
    for (int o = nw >> 1; o > 0; o >>= 1) {
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

// A thread's N vectors of the columns it owns (vector v * tpr + t); zeros
// behind the row.
template <typename T, int VB, int NV>
__device__ __forceinline__ void load_owned(const T *row, long long inner, int tpr, int nvec,
                                           typename RawVec<VB>::type (&raw)[NV])
{
#pragma unroll
    for (int v = 0; v < NV; v++) {
        const int c = v * tpr + static_cast<int>(threadIdx.x);
        raw[v] = typename RawVec<VB>::type{};
        if (c < nvec)
            raw[v] = load_row_vec<T, VB>(row, c, inner);
    }
}

// gamma or beta for the owned columns, as pairs; `none` where it is null.
template <typename T, int VB, int NV, int P>
__device__ __forceinline__ void load_owned_params(const void *p, int is_f32, float none, int tpr,
                                                  int nvec, Float2 (&out)[P])
{
    constexpr int E = VB / sizeof(T);
    float v[2 * P];
#pragma unroll
    for (int k = 0; k < 2 * P; k++)
        v[k] = none;
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int c = k * tpr + static_cast<int>(threadIdx.x);
        if (p && c < nvec) {
            float e[E];
            load_params<T, E>(p, is_f32, static_cast<long long>(c) * E, e);
#pragma unroll
            for (int i = 0; i < E; i++)
                v[k * E + i] = e[i];
        }
    }
#pragma unroll
    for (int k = 0; k < P; k++)
        out[k] = pair(v[2 * k], v[2 * k + 1]);
}

template <typename T, int VB, int NV>
__device__ __forceinline__ void store_owned(T *row, int tpr, int nvec,
                                            const typename RawVec<VB>::type (&raw)[NV])
{
#pragma unroll
    for (int v = 0; v < NV; v++) {
        const int c = v * tpr + static_cast<int>(threadIdx.x);
        if (c < nvec)
            reinterpret_cast<typename RawVec<VB>::type *>(row)[c] = raw[v];
    }
}

template <int P>
__device__ __forceinline__ float sum_pairs(const Float2 (&v)[P])
{
    Float2 s = v[0];
#pragma unroll
    for (int k = 1; k < P; k++)
        s = add2(s, v[k]);
    float lo, hi;
    split(s, lo, hi);
    return lo + hi;
}

// Forwards: blocks walk the rows with a stride of the grid.  The parameters
// are read once and the next row's loads are in flight while the current row's
// two sums are joined.  Arithmetic is on pairs of columns.
template <typename T, int VB, int NV>
__global__ void __launch_bounds__(512) layer_norm_kernel(const LayerNormParams p)
{
    constexpr int E = VB / sizeof(T);
    constexpr int P = (NV * E + 1) / 2;
    using Raw = typename RawVec<VB>::type;
    __shared__ float buf[2][1][32];
    grid_dependency_wait();
    grid_launch_dependents();
    const int tpr = blockDim.x, nvec = p.cols / E;
    const float inv = 1.0f / static_cast<float>(p.cols);
    const long long step = static_cast<long long>(gridDim.x) * blockDim.y;
    const long long first = static_cast<long long>(blockIdx.x) * blockDim.y;
    Raw raw[NV];
    Float2 gam[P], bet[P];
    auto fetch = [&](long long r) {
        if (r < p.rows)
            load_owned<T, VB, NV>(static_cast<const T *>(p.x) + row_offset(p.xv, r), p.x_inner, tpr,
                                  nvec, raw);
    };
    fetch(first + threadIdx.y);
    load_owned_params<T, VB, NV>(p.gamma, p.gamma_f32, 1.0f, tpr, nvec, gam);
    load_owned_params<T, VB, NV>(p.beta, p.beta_f32, 0.0f, tpr, nvec, bet);
    // every group of the block makes the same number of steps
    for (long long base = first; base < p.rows; base += step) {
        const long long r = base + threadIdx.y;
        Float2 x[P];
        unpack_pairs<T, VB>(raw, x);
        fetch(r + step);
        float sum[1] = {sum_pairs(x)};
        group_sum(sum, buf[0], tpr);
        const float mean = sum[0] * inv;
        const Float2 minus = pair(-mean, -mean);
        Float2 sq[2] = {pair(0.0f, 0.0f), pair(0.0f, 0.0f)};
#pragma unroll
        for (int k = 0; k < P; k++)
            x[k] = add2(x[k], minus);
        // columns behind the row hold -mean here: they are left out
#pragma unroll
        for (int k = 0; k < P; k++) {
            if constexpr (E >= 2) {
                if ((k / (E / 2)) * tpr + static_cast<int>(threadIdx.x) < nvec)
                    sq[k & 1] = fma2(x[k], x[k], sq[k & 1]);
            } else {
                float lo, hi;
                split(x[k], lo, hi);
                lo = 2 * k * tpr + static_cast<int>(threadIdx.x) < nvec ? lo : 0.0f;
                hi = 2 * k + 1 < NV && (2 * k + 1) * tpr + static_cast<int>(threadIdx.x) < nvec
                         ? hi : 0.0f;
                const Float2 q = pair(lo, hi);
                sq[k & 1] = fma2(q, q, sq[k & 1]);
            }
        }
        float var[1] = {sum_pairs(sq)};
        group_sum(var, buf[1], tpr);
        if (r >= p.rows)
            continue;
        const float rstd = 1.0f / sqrtf(var[0] * inv + p.eps);
        if (threadIdx.x == 0 && p.mean) {
            p.mean[r] = mean;
            p.rstd[r] = rstd;
        }
        const Float2 scale = pair(rstd, rstd);
#pragma unroll
        for (int k = 0; k < P; k++)
            x[k] = fma2(mul2(x[k], scale), gam[k], bet[k]);
        Raw out[NV];
        pack_pairs<T, VB>(x, out);
        store_owned<T, VB, NV>(static_cast<T *>(p.out) + r * p.cols, tpr, nvec, out);
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
// loads are issued before the current row's sums are joined.  The mean leaves x
// before the product with s: x - m is nearly exact, where m s, rounded
// on its own, would leave an error of the size of |m s| in every column of a
// row that is far from zero.  On pairs of columns, with dx = s a - s mean(a) -
// n s mean(a n), an element costs about eight instructions; in scalar form
// issuing them, not memory, was the bound.
template <typename T, int VB, int NV>
__global__ void __launch_bounds__(512) layer_norm_backward_kernel(const LayerNormParams p)
{
    constexpr int E = VB / sizeof(T);
    constexpr int P = (NV * E + 1) / 2;
    using Raw = typename RawVec<VB>::type;
    __shared__ float buf[2][2][32];
    extern __shared__ float sums[];      // [2][cols] when a block has several groups
    grid_dependency_wait();
    grid_launch_dependents();
    const int tpr = blockDim.x, nvec = p.cols / E;
    const float inv = 1.0f / static_cast<float>(p.cols);
    const long long step = static_cast<long long>(gridDim.x) * blockDim.y;
    const long long first = static_cast<long long>(blockIdx.x) * blockDim.y;
    const Float2 zero = pair(0.0f, 0.0f);
    Raw rx[NV], rg[NV];
    float mean = 0.0f, rstd = 0.0f;
    auto fetch = [&](long long r) {
        if (r < p.rows) {
            load_owned<T, VB, NV>(static_cast<const T *>(p.x) + row_offset(p.xv, r), p.x_inner, tpr,
                                  nvec, rx);
            load_owned<T, VB, NV>(static_cast<const T *>(p.grad) + row_offset(p.gv, r), p.g_inner,
                                  tpr, nvec, rg);
            mean = __ldg(p.mean + r);
            rstd = __ldg(p.rstd + r);
        } else {                         // adds nothing to any sum
#pragma unroll
            for (int v = 0; v < NV; v++)
                rx[v] = rg[v] = Raw{};
            mean = rstd = 0.0f;
        }
    };
    fetch(first + threadIdx.y);
    Float2 gam[P], dg[P], db[P];
    load_owned_params<T, VB, NV>(p.gamma, p.gamma_f32, 1.0f, tpr, nvec, gam);
#pragma unroll
    for (int k = 0; k < P; k++)
        dg[k] = db[k] = zero;
    int parity = 0;
    // every group of the block makes the same number of steps
    for (long long base = first; base < p.rows; base += step, parity ^= 1) {
        const long long r = base + threadIdx.y;
        const float rs = rstd;
        const Float2 rs2 = pair(rs, rs), minus = pair(-mean, -mean);
        Float2 n[P], a[P], s0 = zero, s1 = zero;
        unpack_pairs<T, VB>(rx, n);
        unpack_pairs<T, VB>(rg, a);
        fetch(r + step);
#pragma unroll
        for (int k = 0; k < P; k++) {
            n[k] = mul2(add2(n[k], minus), rs2);
            dg[k] = fma2(a[k], n[k], dg[k]);
            db[k] = add2(db[k], a[k]);
            a[k] = mul2(a[k], gam[k]);
            s0 = add2(s0, a[k]);
            s1 = fma2(a[k], n[k], s1);
        }
        float s[2], hi;
        split(s0, s[0], hi);
        s[0] += hi;
        split(s1, s[1], hi);
        s[1] += hi;
        group_sum(s, buf[parity], tpr);
        if (r >= p.rows)
            continue;
        const float c0 = -s[0] * inv * rs, c1 = -s[1] * inv * rs;
        const Float2 ca = pair(c0, c0), cn = pair(c1, c1);
#pragma unroll
        for (int k = 0; k < P; k++)
            a[k] = fma2(a[k], rs2, fma2(n[k], cn, ca));
        Raw out[NV];
        pack_pairs<T, VB>(a, out);
        store_owned<T, VB, NV>(static_cast<T *>(p.out) + r * p.cols, tpr, nvec, out);
    }
    if (!p.partial)
        return;
    float *part = p.partial + static_cast<long long>(blockIdx.x) * 2 * p.cols;
    float *dst = blockDim.y > 1 ? sums : part;
    for (int y = 0; y < static_cast<int>(blockDim.y); y++) {
        if (static_cast<int>(threadIdx.y) == y) {
            float g[2 * P], b[2 * P];
#pragma unroll
            for (int q = 0; q < P; q++) {
                split(dg[q], g[2 * q], g[2 * q + 1]);
                split(db[q], b[2 * q], b[2 * q + 1]);
            }
#pragma unroll
            for (int v = 0; v < NV; v++) {
                const int c = (v * tpr + static_cast<int>(threadIdx.x)) * E;
                if (c < p.cols) {
#pragma unroll
                    for (int i = 0; i < E; i++) {
                        const float dgi = g[v * E + i], dbi = b[v * E + i];
                        dst[c + i] = y == 0 ? dgi : dst[c + i] + dgi;
                        dst[p.cols + c + i] = y == 0 ? dbi : dst[p.cols + c + i] + dbi;
                    }
                }
            }
        }
        if (blockDim.y > 1)
            __syncthreads();
    }
    if (blockDim.y > 1) {
        const int threads = blockDim.x * blockDim.y;
        for (int c = threadIdx.y * tpr + threadIdx.x; c < 2 * p.cols; c += threads)
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
    part[static_cast<long long>(p.cols) + c] = db;
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
