// Launches of the layer norm kernels (layer_norm.cuh): which vector width,
// how many threads a row, how many blocks.
#include "gemm_sm100.h"

#include "layer_norm.cuh"

#include <algorithm>
#include <cstring>

using namespace ptg;

namespace {

constexpr int kMaxThreads = 512;
constexpr int kBlockThreads = 256;      // a block holds several rows while they are short
constexpr int kBackwardBlocksPerSm = 2;
constexpr int kMaxBackwardBlocks = 512;  // bounds the partial sums whatever the device
constexpr int kLongRowParts = 64;       // row strides of the long-row parameter sums

// A call's first launch, for gemm_sm100_last_launch (the second one adds up the
// partial sums).
thread_local int t_grid = 0, t_block = 0;

template <typename Kernel, typename... Args>
cudaError_t launch(Kernel kernel, dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                   Args... args)
{
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg;
    std::memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (t_grid == 0) {
        t_grid = static_cast<int>(grid.x * grid.y);
        t_block = static_cast<int>(block.x * block.y);
    }
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

bool rows_aligned(const void *p, const RowView &v, int es, int bytes)
{
    if (reinterpret_cast<uintptr_t>(p) % bytes != 0)
        return false;
    for (int d = 0; d < v.n; d++)
        if (v.stride[d] * es % bytes != 0)
            return false;
    return true;
}

// The widest vector (bytes) every row of the call starts aligned to and the
// row length is a multiple of; one element where the last axis is strided.
int vector_bytes(const PtgLayerNorm &a, int es)
{
    if (a.x_inner != 1 || (a.grad && a.g_inner != 1))
        return es;
    for (int vb : {16, 8, 4}) {
        if (vb <= es)
            break;
        if (static_cast<long long>(a.cols) * es % vb != 0)
            continue;
        auto params = [&](const void *p, int f32) {
            return !p || reinterpret_cast<uintptr_t>(p) % (f32 ? 4 : vb) == 0;
        };
        if (rows_aligned(a.x, a.xv, es, vb) && (!a.grad || rows_aligned(a.grad, a.gv, es, vb)) &&
            reinterpret_cast<uintptr_t>(a.out) % vb == 0 && params(a.gamma, a.gamma_f32) &&
            params(a.beta, a.beta_f32))
            return vb;
    }
    return es;
}

// Threads of a row's group: the fewest (a power of two) that hold the row in
// at most `nv` vectors each.
int group_threads(long long nvec, int nv)
{
    int t = 8;
    while (t < kMaxThreads && static_cast<long long>(t) * nv < nvec)
        t *= 2;
    return t;
}

LayerNormParams params_of(const PtgLayerNorm &a)
{
    LayerNormParams p;
    std::memset(&p, 0, sizeof(p));
    p.x = a.x;
    p.grad = a.grad;
    p.gamma = a.gamma;
    p.beta = a.beta;
    p.out = a.out;
    p.mean = a.mean;
    p.rstd = a.rstd;
    p.xv = a.xv;
    p.gv = a.gv;
    p.x_inner = a.x_inner;
    p.g_inner = a.g_inner;
    p.rows = a.rows;
    p.cols = a.cols;
    p.eps = a.eps;
    p.gamma_f32 = a.gamma_f32;
    p.beta_f32 = a.beta_f32;
    return p;
}

// ------------------------------------------------------------ forwards
// Sixteen elements a thread, or 32 where the row is too long for that.  With few
// rows the row is spread over more threads instead (one vector each), which
// shortens the chain of loads that a launch of a few blocks waits for.
template <typename T, int VB>
cudaError_t forward(const LayerNormParams &p, int sms, cudaStream_t stream)
{
    constexpr int E = VB / sizeof(T);
    constexpr int kMost = 32 / E, kUsual = 16 / E;
    const long long nvec = p.cols / E;
    if (nvec > static_cast<long long>(kMost) * kMaxThreads) {
        const long long grid = std::min<long long>(p.rows, sms * 8ll);
        return launch(layer_norm_long_kernel<T>, dim3(static_cast<unsigned>(grid)),
                      dim3(kMaxThreads), 0, stream, p);
    }
    const int tpr = group_threads(nvec, p.rows <= 4ll * sms ? 1 : std::min(kUsual, 8));
    const int nv = static_cast<int>((nvec + tpr - 1) / tpr);
    const dim3 block(tpr, std::max(1, kBlockThreads / tpr));
    const int threads = static_cast<int>(block.x * block.y);
    const long long grid = std::min<long long>((p.rows + block.y - 1) / block.y,
                                               sms * static_cast<long long>(1024 / threads));
    const dim3 g(static_cast<unsigned>(grid));
    if (nv <= 1)
        return launch(layer_norm_kernel<T, VB, 1>, g, block, 0, stream, p);
    if (nv <= 2)
        return launch(layer_norm_kernel<T, VB, 2>, g, block, 0, stream, p);
    if (nv <= 4)
        return launch(layer_norm_kernel<T, VB, 4>, g, block, 0, stream, p);
    if constexpr (kMost > 4) {
        if (nv <= 8)
            return launch(layer_norm_kernel<T, VB, 8>, g, block, 0, stream, p);
        if constexpr (kMost > 8) {
            if (nv <= 16)
                return launch(layer_norm_kernel<T, VB, 16>, g, block, 0, stream, p);
            if constexpr (kMost > 16)
                return launch(layer_norm_kernel<T, VB, 32>, g, block, 0, stream, p);
        }
    }
    return cudaErrorInvalidValue;
}

// ------------------------------------------------------------ backwards
template <typename T, int VB, int NV>
cudaError_t backward_nv(LayerNormParams &p, const PtgLayerNorm &a, int tpr, const PtgDevice &dev,
                        cudaStream_t stream)
{
    const dim3 block(tpr, std::max(1, kBlockThreads / tpr));
    const long long need = (p.rows + block.y - 1) / block.y;
    const int grid = static_cast<int>(
        std::min<long long>(need, std::min(dev.sms * kBackwardBlocksPerSm, kMaxBackwardBlocks)));
    const bool want = a.dgamma || a.dbeta;
    p.partial = want ? a.partial : nullptr;
    const size_t smem = want && block.y > 1 ? static_cast<size_t>(2) * p.cols * 4 : 0;
    cudaError_t err = launch(layer_norm_backward_kernel<T, VB, NV>, dim3(grid), block, smem,
                             stream, p);
    if (err == cudaSuccess && want)
        err = launch(sum_partials_kernel, dim3((p.cols + 31) / 32, 2), dim3(1024), 0, stream,
                     static_cast<const float *>(p.partial), grid, 2ll * p.cols, p.cols, a.dgamma,
                     a.dbeta);
    return err;
}

// Sixteen elements a thread at most: with their gradients' sums and the next
// row's loads that is what 128 registers hold.
template <typename T, int VB>
cudaError_t backward(LayerNormParams &p, const PtgLayerNorm &a, const PtgDevice &dev, cudaStream_t stream)
{
    constexpr int E = VB / sizeof(T);
    constexpr int kMost = 16 / E;
    const long long nvec = p.cols / E;
    if (nvec > static_cast<long long>(kMost) * kMaxThreads) {
        const long long grid = std::min<long long>(p.rows, dev.sms * 8ll);
        cudaError_t err = launch(layer_norm_backward_long_kernel<T>,
                                 dim3(static_cast<unsigned>(grid)), dim3(kMaxThreads), 0, stream,
                                 p);
        if (err != cudaSuccess || !(a.dgamma || a.dbeta))
            return err;
        p.partial = a.partial;
        const int parts = static_cast<int>(std::min<long long>(p.rows, kLongRowParts));
        err = launch(layer_norm_param_long_kernel<T>, dim3((p.cols + 255) / 256, parts), dim3(256),
                     0, stream, p);
        if (err == cudaSuccess)
            err = launch(sum_partials_kernel, dim3((p.cols + 31) / 32, 2), dim3(1024), 0, stream,
                         static_cast<const float *>(p.partial), parts, 2ll * p.cols, p.cols,
                         a.dgamma, a.dbeta);
        return err;
    }
    const int tpr = group_threads(nvec, kMost);
    const int nv = static_cast<int>((nvec + tpr - 1) / tpr);
    if (nv <= 1)
        return backward_nv<T, VB, 1>(p, a, tpr, dev, stream);
    if constexpr (kMost > 1)
        if (nv <= 2)
            return backward_nv<T, VB, 2>(p, a, tpr, dev, stream);
    if constexpr (kMost > 2)
        if (nv <= 4)
            return backward_nv<T, VB, 4>(p, a, tpr, dev, stream);
    if constexpr (kMost > 4)
        if (nv <= 8)
            return backward_nv<T, VB, 8>(p, a, tpr, dev, stream);
    if constexpr (kMost > 8)
        return backward_nv<T, VB, 16>(p, a, tpr, dev, stream);
    return cudaErrorInvalidValue;
}

template <typename T>
cudaError_t dispatch(const PtgLayerNorm &a, const PtgDevice &dev, bool back,
                     cudaStream_t stream)
{
    LayerNormParams p = params_of(a);
    const int vb = vector_bytes(a, sizeof(T));
    if (vb == 16)
        return back ? backward<T, 16>(p, a, dev, stream) : forward<T, 16>(p, dev.sms, stream);
    if (vb == 8)
        return back ? backward<T, 8>(p, a, dev, stream) : forward<T, 8>(p, dev.sms, stream);
    if constexpr (sizeof(T) == 2)
        if (vb == 2)
            return back ? backward<T, 2>(p, a, dev, stream) : forward<T, 2>(p, dev.sms, stream);
    return back ? backward<T, 4>(p, a, dev, stream) : forward<T, 4>(p, dev.sms, stream);
}

cudaError_t run(const PtgLayerNorm &a, bool back, cudaStream_t stream)
{
    PtgDevice dev;
    if (!ptg_device(&dev))
        return cudaErrorNoDevice;
    t_grid = 0;
    cudaError_t err;
    switch (a.dtype) {
    case DTYPE_FLOAT32: err = dispatch<float>(a, dev, back, stream); break;
    case DTYPE_FLOAT16: err = dispatch<__half>(a, dev, back, stream); break;
    case DTYPE_BFLOAT16: err = dispatch<__nv_bfloat16>(a, dev, back, stream); break;
    default: err = cudaErrorInvalidValue; break;
    }
    if (err == cudaSuccess)
        ptg_record_launch(back ? "layer-norm-backward" : "layer-norm", false, a.dtype, t_grid,
                          t_block, 1);
    return err;
}

} // namespace

cudaError_t ptg_layer_norm(const PtgLayerNorm &a, cudaStream_t stream)
{
    return run(a, false, stream);
}

cudaError_t ptg_layer_norm_backward(const PtgLayerNorm &a, cudaStream_t stream)
{
    return run(a, true, stream);
}

// Partial sums of the parameters: one pair of rows for each block.
size_t ptg_layer_norm_partial_bytes(long long rows, int cols)
{
    return static_cast<size_t>(std::min<long long>(rows, kMaxBackwardBlocks)) * 2 * cols *
           sizeof(float);
}
