// Linear layers over groups of rows: which operands TMA can read as they lie,
// which have to be laid out first, and the launches of ragged_gemm.cuh.
#include "gemm_sm100.h"

#include "linear.cuh"
#include "ragged_decode.cuh"
#include "ragged_simt.cuh"

#include <cudaTypedefs.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <mutex>

using namespace ptg;

namespace {

constexpr size_t kAlign = 256;

long long round8(long long n) { return (n + 7) / 8 * 8; }

int element_bytes(int dtype) { return dtype == DTYPE_FLOAT32 ? 4 : 2; }

// ------------------------------------------------------------ workspace
// Hands out pieces of the caller's workspace; with no workspace it only
// counts, so that one plan both sizes and runs a call.
struct Workspace {
    uint8_t *base;
    size_t used;
    void *take(size_t bytes)
    {
        void *p = base ? base + used : nullptr;
        used += (bytes + kAlign - 1) / kAlign * kAlign;
        return p;
    }
};

// ------------------------------------------------------------ launches
template <typename Kernel, typename... Args>
cudaError_t launch(Kernel kernel, dim3 grid, int block, size_t smem, cudaStream_t stream,
                   Args... args)
{
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg;
    std::memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// A rank-5 tiled map; strides in elements of `es` bytes, axes past `rank`
// have extent 1.
bool encode(const PtgDevice &dev, CUtensorMap *map, int dtype, const void *base, int rank,
            const long long *ext, const long long *stride, int box0, int box1, int box2 = 1,
            bool swizzled = true)
{
    if (!dev.encode)
        return false;
    cuuint64_t dims[5], strides[4];
    cuuint32_t box[5] = {static_cast<cuuint32_t>(box0), static_cast<cuuint32_t>(box1),
                         static_cast<cuuint32_t>(box2), 1, 1};
    cuuint32_t steps[5] = {1, 1, 1, 1, 1};
    const cuuint64_t filler = static_cast<cuuint64_t>(round8(ext[0])) * 2;
    for (int i = 0; i < 5; i++) {
        dims[i] = i < rank ? static_cast<cuuint64_t>(ext[i]) : 1;
        if (i > 0)
            strides[i - 1] = i < rank && dims[i] > 1 ? static_cast<cuuint64_t>(stride[i]) * 2 : filler;
    }
    const CUtensorMapDataType type = dtype == DTYPE_FLOAT16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                            : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(dev.encode)(
               map, type, 5, const_cast<void *>(base), dims, strides, box, steps,
               CU_TENSOR_MAP_INTERLEAVE_NONE,
               swizzled ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) ==
           CUDA_SUCCESS;
}

// ------------------------------------------------------------ operands
// A matrix as the product kernels read it: 16-bit, contiguous along one axis,
// 16-byte aligned, `parts` of them for float32.
struct Rows {
    const void *p;
    long long ld;       // elements between rows
    long long part;     // elements between parts
};

struct Weight {
    const void *p;
    bool cols_contiguous;
    long long ld, group, part;
};

bool aligned(const void *p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Whether rows of this view start at multiples of `bytes`.
bool rows_aligned(const void *p, const RowView &v, int es, int bytes)
{
    if (!aligned(p, bytes))
        return false;
    for (int d = 0; d < v.n; d++)
        if (v.ext[d] > 1 && v.stride[d] * es % bytes != 0)
            return false;
    return true;
}

// What a call has decided; `run` is false while it is only being sized.
struct Plan {
    PtgDevice dev;
    cudaStream_t stream;
    Workspace ws;
    bool run;
    cudaError_t err;
    int parts, passes;      // float32: bfloat16 parts and products of them; else 1, 1
    const char *kernel;     // of the last product, for gemm_sm100_last_kernel
    int grid, block, cluster;   // its launch, or the bias gradient's where there is none
    int dtype;
    LayParams lay[2];       // layouts that the next product waits for
    int lays;

    bool ok() const { return err == cudaSuccess; }
    void then(cudaError_t e)
    {
        if (ok())
            err = e;
    }
    void note(unsigned blocks, int threads, int ctas)
    {
        grid = static_cast<int>(blocks);
        block = threads;
        cluster = ctas;
    }
};

// Launches the layouts asked for so far, two in one launch, with blocks for
// each in proportion to its work: two items a thread as far as five blocks an SM,
// all that fit, go.
void flush_layouts(Plan &pl)
{
    if (pl.lays == 0 || !pl.run || !pl.ok())
        return;
    auto blocks = [&](const LayParams &p) {
        return (p.rows * (p.ld / 8) + 511) / 512;
    };
    const long long n0 = blocks(pl.lay[0]), n1 = pl.lays > 1 ? blocks(pl.lay[1]) : 0;
    const double fit = std::min(1.0, pl.dev.sms * 5.0 / std::max<double>(1.0, n0 + n1));
    const int first = static_cast<int>(std::ceil(n0 * fit)),
              second = static_cast<int>(std::ceil(n1 * fit));
    pl.lays = 0;
    if (first + second == 0)
        return;
    if (pl.dtype == DTYPE_FLOAT32)
        pl.then(launch(lay_out_kernel<float>, dim3(first + second), 256, 0, pl.stream, pl.lay[0],
                       pl.lay[1], first));
    else       // a copy of 16-bit values
        pl.then(launch(lay_out_kernel<__half>, dim3(first + second), 256, 0, pl.stream, pl.lay[0],
                       pl.lay[1], first));
}

// Asks for the layout of `rows` rows of `cols` columns.
void lay_out(Plan &pl, const void *src, const RowView &v, long long inner, long long rows,
             int cols, void *out)
{
    if (pl.lays == 2)
        flush_layouts(pl);
    LayParams &p = pl.lay[pl.lays++];
    std::memset(&p, 0, sizeof(p));
    p.src = src;
    p.rows_of = v;
    p.inner = inner;
    p.rows = rows;
    p.cols = cols;
    p.ld = static_cast<int>(round8(cols));
    p.out = static_cast<uint16_t *>(out);
    p.part = rows * p.ld;
    p.parts = pl.parts;
    p.vec = inner == 1 && rows_aligned(src, v, element_bytes(pl.dtype), 16);
}

// Rows as they lie if TMA can read them, else laid out in the workspace.
Rows plan_rows(Plan &pl, int dtype, const void *p, const RowView &v, long long inner,
               long long rows, int cols)
{
    Rows r;
    r.part = 0;
    if (dtype != DTYPE_FLOAT32 && v.n == 1 && (inner == 1 || cols == 1) &&
        (rows == 1 || v.stride[0] > 0) && rows_aligned(p, v, 2, 16)) {
        r.p = p;
        r.ld = rows == 1 ? round8(cols) : v.stride[0];
        return r;
    }
    r.ld = round8(cols);
    r.part = rows * r.ld;
    void *out = pl.ws.take(static_cast<size_t>(r.part) * pl.parts * 2);
    r.p = out;
    if (pl.run && pl.ok())
        lay_out(pl, p, v, inner, rows, cols, out);
    return r;
}

// Whether the weight can be read as it lies; describes it in *w if so.
bool weight_fits(const PtgLinear &a, Weight *w)
{
    if (a.dtype == DTYPE_FLOAT32 || !aligned(a.w, 16) ||
        !(a.groups == 1 || (a.w_group % 8 == 0 && a.w_group > 0)))
        return false;
    const bool c = (a.w_cols == 1 || a.cols == 1) &&
                   (a.inner == 1 || (a.w_inner % 8 == 0 && a.w_inner > 0));
    const bool k = (a.w_inner == 1 || a.inner == 1) &&
                   (a.cols == 1 || (a.w_cols % 8 == 0 && a.w_cols > 0));
    if (w && (c || k)) {
        w->p = a.w;
        w->cols_contiguous = c;
        w->ld = c ? (a.inner == 1 ? round8(a.cols) : a.w_inner)
                  : (a.cols == 1 ? round8(a.inner) : a.w_cols);
        w->group = a.w_group;
    }
    return c || k;
}

Weight plan_weight(Plan &pl, const PtgLinear &a)
{
    Weight w;
    w.part = 0;
    if (weight_fits(a, &w))
        return w;
    const bool cols_first = a.w_cols == 1 || a.cols == 1;
    const bool inner_first = a.w_inner == 1 || a.inner == 1;
    // laid out along the axis that is contiguous, or else the shorter stride
    w.cols_contiguous = cols_first || (!inner_first && a.w_cols <= a.w_inner);
    const int rows = w.cols_contiguous ? a.inner : a.cols;
    const int cols = w.cols_contiguous ? a.cols : a.inner;
    RowView v;
    std::memset(&v, 0, sizeof(v));
    v.n = 2;
    v.ext[0] = a.groups;
    v.stride[0] = a.groups > 1 ? a.w_group : 0;
    v.ext[1] = rows;
    v.stride[1] = w.cols_contiguous ? a.w_inner : a.w_cols;
    w.ld = round8(cols);
    w.group = rows * w.ld;
    w.part = w.group * a.groups;
    void *out = pl.ws.take(static_cast<size_t>(w.part) * pl.parts * 2);
    w.p = out;
    if (pl.run && pl.ok())
        lay_out(pl, a.w, v, w.cols_contiguous ? a.w_cols : a.w_inner,
                static_cast<long long>(a.groups) * rows, cols, out);
    return w;
}

// By family (pair, few rows, CUDA cores) and type.
const char *kernel_name(int family, int dtype)
{
    static const char *const names[3][3] = {
        {"ragged2-bf16x3-256x256", "ragged2-f16-256x256", "ragged2-bf16-256x256"},
        {"", "ragged-f16-128x64", "ragged-bf16-128x64"},
        {"ragged-simt-f32", "ragged-simt-f16", "ragged-simt-bf16"}};
    return names[family][dtype == DTYPE_FLOAT32 ? 0 : dtype == DTYPE_FLOAT16 ? 1 : 2];
}

// ------------------------------------------------------------ products
constexpr int kMaxDevices = 64;

// The thread's kernel path as far as these layers have it: 1 few rows, 2 CUDA
// cores, 3 pairs; the others are the matmul's own and leave the choice automatic.
int layer_path()
{
    const int path = ptg_path();
    return path <= 3 ? path : 0;
}

// CTA pairs of `kernel` that fit the device at one time; raises its
// shared-memory limit on the first call on a device.  0 on failure.  (The
// kernel is a template argument: the kernels share one function type.)
template <auto kernel>
int pair_count(int sms)
{
    static std::mutex mutex;
    static int counts[kMaxDevices] = {};
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device >= kMaxDevices)
        return 0;
    std::lock_guard<std::mutex> lock(mutex);
    if (counts[device])
        return counts[device];
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRaggedSmem) !=
        cudaSuccess)
        return 0;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg;
    std::memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(static_cast<unsigned>(sms & ~1));
    cfg.blockDim = dim3(kRaggedThreads);
    cfg.dynamicSmemBytes = kRaggedSmem;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) {
        (void)cudaGetLastError();
        n = sms / 2;
    }
    return counts[device] = n;
}

template <typename T, bool INNER, bool CHUNKED>
cudaError_t launch_pairs(Plan &pl, const RaggedMaps &maps, RaggedParams &p, long long bound)
{
    constexpr auto kernel = ragged_gemm_kernel<T, INNER, CHUNKED>;
    const int pairs = pair_count<kernel>(pl.dev.sms);
    if (pairs < 1)
        return cudaErrorInvalidConfiguration;
    p.status = pl.dev.status;
    if (bound > 0x7fffffffll)
        return cudaErrorInvalidValue;
    const long long n = std::max<long long>(1, std::min<long long>(bound, pairs));
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg;
    std::memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(static_cast<unsigned>(2 * n));
    cfg.blockDim = dim3(kRaggedThreads);
    cfg.dynamicSmemBytes = kRaggedSmem;
    cfg.stream = pl.stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    pl.note(cfg.gridDim.x, kRaggedThreads, 2);
    return cudaLaunchKernelEx(&cfg, kernel, maps, p);
}

// Instruction descriptor without its N field.
uint32_t instruction(int dtype, bool a_mn, bool b_mn, int m)
{
    const uint32_t fmt = dtype == DTYPE_FLOAT16 ? 0 : 1;
    return (1u << 4) | (fmt << 7) | (fmt << 10) | (static_cast<uint32_t>(a_mn) << 15) |
           (static_cast<uint32_t>(b_mn) << 16) | (static_cast<uint32_t>(m >> 4) << 24);
}

// The few-row kernel: how many CTAs share the inner axis of a tile.  As many
// as keep two CTAs on every SM, and at least four k-blocks for each.
template <typename T>
cudaError_t launch_decode(Plan &pl, const RaggedMaps &maps, RaggedParams &p)
{
    constexpr auto kernel = ragged_decode_kernel<T>;
    static std::mutex mutex;
    static bool ready[kMaxDevices] = {};
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device >= kMaxDevices)
        return cudaErrorInvalidDevice;
    {
        std::lock_guard<std::mutex> lock(mutex);
        if (!ready[device]) {
            const cudaError_t err = cudaFuncSetAttribute(
                kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, decode_smem(kMaxGroups));
            if (err != cudaSuccess)
                return err;
            ready[device] = true;
        }
    }
    p.status = pl.dev.status;
    const long long tiles = static_cast<long long>((p.features + 127) / 128) *
                            (p.ends ? p.rows / kDecodeRows + std::min(p.groups, p.rows)
                                    : (p.rows + kDecodeRows - 1) / kDecodeRows);
    const int blocks = (p.inner + 63) / 64;
    int split = 1;
    while (split < 8 && tiles * split * 2 <= 2 * pl.dev.sms && blocks >= split * 2 * 4)
        split *= 2;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(split);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg;
    std::memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(static_cast<unsigned>(tiles * split));
    cfg.blockDim = dim3(kDecodeThreads);
    cfg.dynamicSmemBytes = decode_smem(p.ends ? p.groups : 0);
    cfg.stream = pl.stream;
    cfg.attrs = attr;
    cfg.numAttrs = split > 1 ? 2 : 1;
    pl.note(cfg.gridDim.x, kDecodeThreads, split);
    return cudaLaunchKernelEx(&cfg, kernel, maps, p, split);
}

// Few rows: at most a quarter of a tile's on average, or two tiles' when the
// pair kernel would not occupy the GPU once.  Measured on B200 (us, few rows /
// pairs, weights from memory): one 4096 x 4096 weight, 16 rows 11 / 22, 64 rows 14 /
// 23, 128 rows 18 / 23, 256 rows 27 / 24; 32 experts of 2048 x 1024, 32 rows 20 / 28,
// 1024 rows 36 / 31.
bool few_rows(const PtgDevice &dev, long long pair_tiles, int rows, int groups)
{
    return rows <= kDecodeRows / 4 * static_cast<long long>(groups) ||
           (pair_tiles < dev.sms / 2 && rows <= kDecodeRows * 2ll * groups);
}

// ------------------------------------------------------------ CUDA cores
constexpr int kSimtFewRows = 16;

template <typename T, typename TZ, bool INNER, int TF, int TR>
cudaError_t launch_simt_tile(Plan &pl, RaggedSimtParams &s)
{
    constexpr auto kernel = ragged_simt_kernel<T, TZ, INNER, TF, TR>;
    static std::mutex mutex;
    static bool ready[kMaxDevices] = {};
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device >= kMaxDevices)
        return cudaErrorInvalidDevice;
    {
        std::lock_guard<std::mutex> lock(mutex);
        if (!ready[device]) {
            const cudaError_t err =
                cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     ragged_simt_smem<TF, TR>(kMaxGroups));
            if (err != cudaSuccess)
                return err;
            ready[device] = true;
        }
    }
    const RaggedParams &p = s.p;
    const long long row_tiles =
        INNER ? static_cast<long long>((p.cols + TR - 1) / TR) * p.groups
              : (p.ends ? p.rows / TR + std::min(p.groups, p.rows) : (p.rows + TR - 1) / TR);
    const long long tiles = row_tiles * ((p.features + TF - 1) / TF);
    const int steps = ((INNER ? p.rows / p.groups : p.inner) + kSimtStep - 1) / kSimtStep;
    s.split = 1;
    while (s.split < 8 && tiles * s.split * 2 <= 4 * pl.dev.sms && steps >= s.split * 2 * 2)
        s.split *= 2;
    if (tiles * s.split > 2147483647ll)
        return cudaErrorInvalidValue;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(s.split);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg;
    std::memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(static_cast<unsigned>(tiles * s.split));
    cfg.blockDim = dim3(kSimtThreads);
    cfg.dynamicSmemBytes = ragged_simt_smem<TF, TR>(p.ends ? p.groups : 0);
    cfg.stream = pl.stream;
    cfg.attrs = attr;
    cfg.numAttrs = s.split > 1 ? 2 : 1;
    pl.note(cfg.gridDim.x, kSimtThreads, s.split);
    return cudaLaunchKernelEx(&cfg, kernel, s);
}

template <typename T, typename TZ, bool INNER>
cudaError_t launch_simt_rows(Plan &pl, RaggedSimtParams &s)
{
    const int rows = INNER ? s.p.cols : (s.p.rows + s.p.groups - 1) / s.p.groups;
    return rows <= kSimtFewRows ? launch_simt_tile<T, TZ, INNER, 128, 16>(pl, s)
                                : launch_simt_tile<T, TZ, INNER, 64, 64>(pl, s);
}

template <bool INNER>
cudaError_t launch_simt(Plan &pl, RaggedSimtParams &s, int dtype, bool z_f32)
{
    switch (dtype) {
    case DTYPE_FLOAT16:
        return z_f32 ? launch_simt_rows<__half, float, INNER>(pl, s)
                     : launch_simt_rows<__half, __half, INNER>(pl, s);
    case DTYPE_BFLOAT16:
        return z_f32 ? launch_simt_rows<__nv_bfloat16, float, INNER>(pl, s)
                     : launch_simt_rows<__nv_bfloat16, __nv_bfloat16, INNER>(pl, s);
    default: return launch_simt_rows<float, float, INNER>(pl, s);
    }
}

// A matrix of rows with one stride each, in the operands' own type.
struct Plain {
    const void *p;
    long long row, inner;
    bool f32;           // float32 whatever the operands' type (a gradient's dz)
};

// Rows x weight as product() does it.
cudaError_t simt_product(Plan &pl, const PtgLinear &a, const Plain &x, bool transposed,
                         RaggedParams &p)
{
    pl.kernel = kernel_name(2, a.dtype);
    RaggedSimtParams s;
    std::memset(&s, 0, sizeof(s));
    p.ends = a.ends;
    p.groups = a.groups;
    p.rows = a.rows;
    p.features = transposed ? a.inner : a.cols;
    p.inner = transposed ? a.cols : a.inner;
    p.out_row = p.features;
    s.p = p;
    s.a = x.p;
    s.a_row = x.row;
    s.a_inner = x.inner;
    s.b = a.w;
    s.b_inner = transposed ? a.w_cols : a.w_inner;
    s.b_col = transposed ? a.w_inner : a.w_cols;
    s.b_group = a.w_group;
    return launch_simt<false>(pl, s, a.dtype, x.f32);
}

// dw as weight_product() does it.
cudaError_t simt_weight_product(Plan &pl, const PtgLinear &a, const Plain &x,
                                const Plain &dz)
{
    pl.kernel = kernel_name(2, a.dtype);
    RaggedSimtParams s;
    std::memset(&s, 0, sizeof(s));
    s.p.ends = a.ends;
    s.p.groups = a.groups;
    s.p.rows = a.rows;
    s.p.features = a.cols;
    s.p.cols = a.inner;
    s.p.out = a.dw;
    s.p.out_row = a.cols;
    s.p.out_group = static_cast<long long>(a.inner) * a.cols;
    s.out_f32 = a.dw_dtype == DTYPE_FLOAT32;
    s.a = x.p;
    s.a_row = x.inner;
    s.a_inner = x.row;
    s.b = dz.p;
    s.b_inner = dz.row;
    s.b_col = dz.inner;
    return launch_simt<true>(pl, s, a.dtype, dz.f32);
}

// A view's own rows, or a contiguous copy where they have no single stride.
Plain plan_plain(Plan &pl, int dtype, const void *src, const RowView &v, long long inner,
                 long long rows, int cols)
{
    if (v.n == 1)
        return {src, v.stride[0], inner, false};
    void *out = pl.ws.take(static_cast<size_t>(rows) * cols * element_bytes(dtype));
    if (pl.run && pl.ok()) {
        const long long blocks = (rows * cols + 255) / 256;
        const dim3 grid(static_cast<unsigned>(std::min<long long>(blocks, pl.dev.sms * 16ll)));
        if (dtype == DTYPE_FLOAT32)
            pl.then(launch(copy_rows_kernel<float>, grid, 256, 0, pl.stream,
                           static_cast<const float *>(src), v, inner, rows, cols,
                           static_cast<float *>(out)));
        else
            pl.then(launch(copy_rows_kernel<uint16_t>, grid, 256, 0, pl.stream,
                           static_cast<const uint16_t *>(src), v, inner, rows, cols,
                           static_cast<uint16_t *>(out)));
    }
    return {out, cols, 1, false};
}

// ------------------------------------------------------------ tensor cores
// Maps of a 16-bit result (and of pre), where TMA can store to them.
void result_maps(const Plan &pl, int dtype, RaggedParams &p, RaggedMaps &maps, long long rows,
                 int groups)
{
    if (dtype == DTYPE_FLOAT32 || p.features % 8 != 0 || !aligned(p.out, 16) ||
        (p.pre && !aligned(p.pre, 16)))
        return;
    const long long ext[3] = {p.features, rows, groups};
    const long long str[3] = {1, p.out_row, p.out_group};
    p.tma_store =
        encode(pl.dev, &maps.out, dtype, p.out, 3, ext, str, 32, kGroup, 1, false) &&
        (!p.pre || encode(pl.dev, &maps.pre, dtype, p.pre, 3, ext, str, 32, kGroup, 1, false));
}

// Rows x weight: `features` columns of the result, `inner` summed over.
// transposed: the weight's inner axis gives the features (dx).
cudaError_t product(Plan &pl, const PtgLinear &a, const Rows &x, const Weight &w,
                    bool transposed, RaggedParams &p)
{
    const int features = transposed ? a.inner : a.cols, inner = transposed ? a.cols : a.inner;
    p.ends = a.ends;
    p.groups = a.groups;
    p.rows = a.rows;
    p.features = features;
    p.inner = inner;
    p.a_mn = transposed ? !w.cols_contiguous : w.cols_contiguous;
    p.passes = pl.passes;
    p.parts = pl.parts;
    p.out_row = features;
    RaggedMaps maps;
    std::memset(&maps, 0, sizeof(maps));
    p.a_chunks = p.a_mn && features % 64 == 0;
    const long long wext[5] = {p.a_chunks ? 64 : p.a_mn ? features : inner,
                               p.a_mn ? inner : features,
                               p.a_chunks ? features / 64 : a.groups,
                               p.a_chunks ? a.groups : pl.parts, pl.parts};
    const long long wstr[5] = {1, w.ld, p.a_chunks ? 64 : w.group, p.a_chunks ? w.group : w.part,
                               w.part};
    const long long xext[3] = {inner, a.rows, pl.parts};
    const long long xstr[3] = {1, x.ld, x.part};
    if (inner > 0) {
        bool ok = encode(pl.dev, &maps.a, a.dtype, w.p, p.a_chunks ? 5 : 4, wext, wstr, 64,
                         p.a_mn ? 64 : 128, p.a_chunks ? 2 : 1);
        for (int i = 0; i < 4; i++)
            ok = ok && encode(pl.dev, &maps.rows[i], a.dtype, x.p, 3, xext, xstr, 64, 16 << i);
        if (!ok)
            return cudaErrorInvalidValue;
    }
    p.split = 1;
    const long long ft = (features + 255) / 256;
    auto row_tiles = [&](int span) {
        return a.ends ? a.rows / span + std::min(a.groups, a.rows)
                      : static_cast<long long>((a.rows + span - 1) / span);
    };
    // tiles of fewer rows while the pairs are not all at work: they load more
    // of the weight per row, but an idle pair loads nothing (us, so / in tiles of
    // 256 rows: 256 x 4096 x 4096 23.1 / 26.4, 512 x 4096 x 1024 22.2 / 26.2,
    // float32 4698 x 2816 x 102 149 / 171)
    p.span = kRaggedBN;
    long long bound = ft * row_tiles(p.span);
    const int path = layer_path();
    const bool few = a.dtype != DTYPE_FLOAT32 && path != 3 &&
                     (path == 1 || few_rows(pl.dev, bound, a.rows, a.groups));
    p.idesc = instruction(a.dtype, p.a_mn, false, few ? 128 : 256);
    pl.kernel = kernel_name(few ? 1 : 0, a.dtype);
    flush_layouts(pl);
    if (!pl.ok())
        return pl.err;
    while (p.span > 64 && ft * row_tiles(p.span / 2) <= pl.dev.sms / 2) {
        p.span /= 2;
        bound = ft * row_tiles(p.span);
    }
    if (few)
        return a.dtype == DTYPE_FLOAT16 ? launch_decode<__half>(pl, maps, p)
                                        : launch_decode<__nv_bfloat16>(pl, maps, p);
    result_maps(pl, a.dtype, p, maps, a.rows, 1);
    switch (a.dtype) {
    case DTYPE_FLOAT16: return launch_pairs<__half, false, false>(pl, maps, p, bound);
    case DTYPE_BFLOAT16: return launch_pairs<__nv_bfloat16, false, false>(pl, maps, p, bound);
    default: return launch_pairs<float, false, true>(pl, maps, p, bound);
    }
}

// Parts that the rows of a group are cut into for dw: while its tiles leave
// pairs idle, and every part keeps eight k-blocks on average (us, so / in one
// part: 16026 rows, 384 x 112 17.2 / 77.3; 4096 rows, 512 x 512 13.2 / 25.5; 8192
// rows, 1024 x 1024 21.7 / 43.5).  A rule of the sizes alone, since it also sizes
// the workspace.
constexpr int kPairs = 74;

int weight_parts(const PtgLinear &a)
{
    const long long tiles = static_cast<long long>((a.cols + 255) / 256) *
                            ((a.inner + kRaggedBN - 1) / kRaggedBN) * a.groups;
    const long long blocks = a.rows / a.groups / 64;
    return static_cast<int>(std::max<long long>(1, std::min(kPairs / tiles, blocks / 8)));
}

// dw[g] = sum over the rows of group g of x^T dz.  With several parts each
// writes its float32 sums to `partial`, and add_parts_kernel joins them.
cudaError_t weight_product(Plan &pl, const PtgLinear &a, const Rows &x, const Rows &dz,
                           CUtensorMap *group_maps, int parts, float *partial)
{
    pl.kernel = kernel_name(0, a.dtype);
    flush_layouts(pl);
    if (!pl.ok())
        return pl.err;
    RaggedParams p;
    std::memset(&p, 0, sizeof(p));
    p.ends = a.ends;
    p.groups = a.groups;
    p.rows = a.rows;
    p.features = a.cols;
    p.cols = a.inner;
    p.passes = pl.passes;
    p.parts = pl.parts;
    p.span = kRaggedBN;
    p.split = parts;
    p.idesc = instruction(a.dtype, true, true, 256);
    p.out = parts > 1 ? partial : a.dw;
    p.out_row = a.cols;
    p.out_group = static_cast<long long>(a.inner) * a.cols;
    p.out_part = p.out_group * a.groups;
    RaggedMaps maps;
    std::memset(&maps, 0, sizeof(maps));
    auto rows_map = [&](CUtensorMap *map, const Rows &m, int cols, int chunks) {
        const long long ext[4] = {chunks ? 64 : cols, a.rows, chunks ? cols / 64 : pl.parts,
                                  pl.parts};
        const long long str[4] = {1, m.ld, chunks ? 64 : m.part, m.part};
        return encode(pl.dev, map, a.dtype, m.p, chunks ? 4 : 3, ext, str, 64, 64, chunks ? 2 : 1);
    };
    p.a_chunks = a.cols % 64 == 0;
    p.b_chunks = a.inner % 64 == 0;
    if (!rows_map(&maps.a, dz, a.cols, p.a_chunks) || !rows_map(&maps.b, x, a.inner, p.b_chunks))
        return cudaErrorInvalidValue;
    cudaError_t err = cudaSuccess;
    if (a.ends) {
        p.group_maps = group_maps;
        err = launch(group_maps_kernel, dim3(1), 256, static_cast<size_t>(a.groups) * 8, pl.stream,
                     maps.a, maps.b, a.ends, a.groups, a.rows, group_maps);
        if (err != cudaSuccess)
            return err;
    }
    const long long bound = static_cast<long long>((a.cols + 255) / 256) *
                            ((a.inner + kRaggedBN - 1) / kRaggedBN) * a.groups * parts;
    const int out_dtype = parts > 1 ? static_cast<int>(DTYPE_FLOAT32) : a.dw_dtype;
    result_maps(pl, out_dtype, p, maps, a.inner, a.groups);
    if (a.dtype == DTYPE_FLOAT32)
        err = launch_pairs<float, true, true>(pl, maps, p, bound);
    else if (out_dtype == DTYPE_FLOAT32)
        err = launch_pairs<float, true, false>(pl, maps, p, bound);
    else if (a.dtype == DTYPE_FLOAT16)
        err = launch_pairs<__half, true, false>(pl, maps, p, bound);
    else
        err = launch_pairs<__nv_bfloat16, true, false>(pl, maps, p, bound);
    if (err != cudaSuccess || parts == 1)
        return err;
    const long long n = p.out_part;
    const int vec = n % 4 == 0 && aligned(a.dw, 16);
    const dim3 grid(static_cast<unsigned>(
        std::min<long long>((n + 1023) / 1024, pl.dev.sms * 16ll)));
    if (a.dw_dtype == DTYPE_FLOAT32)
        return launch(add_parts_kernel<float>, grid, 256, 0, pl.stream,
                      static_cast<const float *>(partial), parts, n, n, vec,
                      static_cast<float *>(a.dw));
    if (a.dw_dtype == DTYPE_FLOAT16)
        return launch(add_parts_kernel<__half>, grid, 256, 0, pl.stream,
                      static_cast<const float *>(partial), parts, n, n, vec,
                      static_cast<__half *>(a.dw));
    return launch(add_parts_kernel<__nv_bfloat16>, grid, 256, 0, pl.stream,
                  static_cast<const float *>(partial), parts, n, n, vec,
                  static_cast<__nv_bfloat16 *>(a.dw));
}

bool begin(Plan &pl, const PtgLinear &a, bool run, cudaStream_t stream)
{
    std::memset(&pl, 0, sizeof(pl));
    pl.err = cudaSuccess;
    pl.stream = stream;
    pl.dtype = a.dtype;
    pl.run = run;
    if (run && a.workspace)
        pl.ws.base = reinterpret_cast<uint8_t *>(
            (reinterpret_cast<uintptr_t>(a.workspace) + kAlign - 1) / kAlign * kAlign);
    const bool split = a.dtype == DTYPE_FLOAT32;
    const bool tf32 = ptg_precision() == CUDA_MATMUL_PRECISION_TF32;
    pl.parts = !split ? 1 : tf32 ? 2 : 3;
    pl.passes = !split ? 1 : tf32 ? 3 : 6;
    return !run || ptg_device(&pl.dev);
}

// Whether a product runs on the CUDA cores: float32 ones below kSimtWork
// multiply-adds, 16-bit ones below kSimtLayWork whose operands would have to
// be laid out first.  The bound lies where the two cross for weights of a million
// elements; measured on B200 (us, CUDA cores / three parts on the tensor cores): 64 x
// 1024 x 1024 15 / 37, 512 x 1024 x 1024 49 / 41, 1024 x 1024 x 1024 90 / 43; 16 experts of
// 1024 x 1024, 256 rows 64 / 88, 2048 rows 213 / 108.  For larger weights, whose parts
// the tensor cores' path writes and reads again on every call, they cross at more work
// than the bound, and between the two it takes the slower side: 8 x 4096 x 4096 38 /
// 139 (CUDA cores), but 64 x 4096 x 4096 89 / 144, 8 x 8192 x 8192 142 / 341 and 64 experts
// of 2048 x 1408 with 2048 rows 782 / 834 (tensor cores).  The thread's kernel path
// decides first (2: CUDA cores, 1 and 3: the tensor-core kernels).
constexpr double kSimtWork = 5.0e8;
constexpr double kSimtLayWork = 5.0e7;

// Elements of dz up to which 16-bit operands with an activation keep it in
// float32, and so take the CUDA cores.  Rounding dz puts the gradients at 1.2 units
// of roundoff from float64 in the norm, at any size, instead of 0.85; in
// sums of a few terms nothing averages out (one row: dw's worst element 45
// instead of 24 units of its rms).  us, float32 / rounded on the tensor cores, both
// gradients: 64 x 1024 x 256 28 / 33, 16 x 1024 x 1024 28 / 20, 16 x 4096 x 1024 62 / 22,
// 4 x 4096 x 4096 155 / 29: up to here the exact form costs some 20 us for layers
// of ordinary width, and a wide layer's few rows pay in proportion to its weight.
constexpr double kExactGradient = 16384;

bool on_cuda_cores(const PtgLinear &a, bool lay)
{
    const int path = layer_path();
    if (path == 1 || path == 3)
        return false;
    const double work = static_cast<double>(a.rows) * a.inner * a.cols;
    if (path == 2)
        return true;
    return a.dtype == DTYPE_FLOAT32 ? work <= kSimtWork : lay && work <= kSimtLayWork;
}

// Whether the tensor-core kernels would need this call's operands laid out.
bool needs_layout(const PtgLinear &a, const void *rows, const RowView &v, long long inner, int cols)
{
    const bool rows_fit = v.n == 1 && (inner == 1 || cols == 1) &&
                          (a.rows == 1 || v.stride[0] > 0) && rows_aligned(rows, v, 2, 16);
    return !rows_fit || !weight_fits(a, nullptr);
}

void forward(Plan &pl, const PtgLinear &a)
{
    RaggedParams p;
    std::memset(&p, 0, sizeof(p));
    p.act = a.activation;
    p.out = a.y;
    p.pre = a.pre;
    p.bias = a.bias;
    p.bias_f32 = a.bias_f32;
    if (a.residual) {
        const Plain r =
            plan_plain(pl, a.dtype, a.residual, a.rv, a.r_inner, a.rows, a.cols);
        p.residual = r.p;
        p.residual_row = r.row;
        p.residual_inner = r.inner;
        p.residual_small = static_cast<double>(a.rows) * std::max(1ll, r.row) +
                               static_cast<double>(a.cols) * r.inner <
                           2147483648.0 / element_bytes(a.dtype);
    }
    if (on_cuda_cores(a, needs_layout(a, a.x, a.xv, a.x_inner, a.inner))) {
        const Plain x = plan_plain(pl, a.dtype, a.x, a.xv, a.x_inner, a.rows, a.inner);
        if (pl.run && pl.ok())
            pl.then(simt_product(pl, a, x, false, p));
        return;
    }
    const Rows x = plan_rows(pl, a.dtype, a.x, a.xv, a.x_inner, a.rows, a.inner);
    const Weight w = plan_weight(pl, a);
    if (pl.run && pl.ok())
        pl.then(product(pl, a, x, w, false, p));
}

// Launches slope_kernel and, for dbias, group_sums_kernel; `parts` 0 leaves dz
// in float32.
void slope(Plan &pl, const PtgLinear &a, void *dz, int parts, float *partial)
{
    SlopeParams p;
    std::memset(&p, 0, sizeof(p));
    const int es = element_bytes(a.dtype);
    p.grad = a.grad;
    p.pre = a.pre;
    p.gv = a.gv;
    p.pv = a.pv;
    p.g_inner = a.g_inner;
    p.p_inner = a.p_inner;
    p.ends = a.ends;
    p.groups = a.groups;
    p.rows = a.rows;
    p.cols = a.cols;
    p.act = a.activation;
    p.g_vec = a.g_inner == 1 && rows_aligned(a.grad, a.gv, es, 16);
    p.p_vec = a.p_inner == 1 && rows_aligned(a.pre, a.pv, es, 16);
    p.dz = dz;
    p.ld = static_cast<int>(round8(a.cols));
    p.part = static_cast<long long>(a.rows) * p.ld;
    p.parts = parts;
    p.partial = partial;
    p.strips = (a.cols + kSlopeCols - 1) / kSlopeCols;
    const dim3 grid(static_cast<unsigned>(p.strips) *
                    (a.rows / kSlopeRows + std::min(a.groups, a.rows)));
    const size_t table = static_cast<size_t>(a.groups) * 8;
    pl.note(grid.x, 256, 1);
    switch (a.dtype) {
    case DTYPE_FLOAT16: pl.then(launch(slope_kernel<__half>, grid, 256, table, pl.stream, p)); break;
    case DTYPE_BFLOAT16:
        pl.then(launch(slope_kernel<__nv_bfloat16>, grid, 256, table, pl.stream, p));
        break;
    default: pl.then(launch(slope_kernel<float>, grid, 256, table, pl.stream, p)); break;
    }
    if (partial && pl.ok())
        pl.then(launch(group_sums_kernel, dim3((a.cols + 31) / 32, a.groups), 1024, table,
                       pl.stream, static_cast<const float *>(partial), a.ends, a.groups, a.rows,
                       a.cols, a.dbias));
}

void backward(Plan &pl, const PtgLinear &a)
{
    const bool active = a.activation != CUDA_MATMUL_EPILOGUE_NONE;
    const bool products = a.dx || a.dw;
    const bool lay = (!active && needs_layout(a, a.grad, a.gv, a.g_inner, a.cols)) ||
                     needs_layout(a, a.x, a.xv, a.x_inner, a.inner);
    // dz of a few rows stays in float32: below some thousand elements its
    // roundings to 16 bits would not average out in the products
    const bool exact = a.dtype != DTYPE_FLOAT32 && active &&
                       static_cast<double>(a.rows) * a.cols <= kExactGradient;
    const bool simt = on_cuda_cores(a, lay) || (exact && layer_path() == 0);
    const size_t partial_rows = a.rows / kSlopeRows + std::min(a.groups, a.rows);
    float *partial = a.dbias ? static_cast<float *>(pl.ws.take(partial_rows * a.cols * 4)) : nullptr;

    // dz in the form that the products read.  float32 on the tensor cores goes
    // through slope_kernel without an activation too: it then lays out grad's
    // parts and sums its columns in one pass.
    Rows dz;
    Plain plain;
    std::memset(&dz, 0, sizeof(dz));
    std::memset(&plain, 0, sizeof(plain));
    if (products && (active || (a.dtype == DTYPE_FLOAT32 && !simt))) {
        dz.ld = round8(a.cols);
        dz.part = a.rows * dz.ld;
        const size_t each = simt ? 4 : 2 * static_cast<size_t>(pl.parts);
        void *out = pl.ws.take(static_cast<size_t>(dz.part) * each);
        dz.p = out;
        plain = {out, dz.ld, 1, true};
        if (pl.run && pl.ok())
            slope(pl, a, out, simt ? 0 : pl.parts, partial);
    } else {
        if (products && simt)
            plain = plan_plain(pl, a.dtype, a.grad, a.gv, a.g_inner, a.rows, a.cols);
        else if (products)
            dz = plan_rows(pl, a.dtype, a.grad, a.gv, a.g_inner, a.rows, a.cols);
        if (a.dbias && pl.run && pl.ok())
            slope(pl, a, nullptr, 0, partial);
    }
    RaggedParams p;
    std::memset(&p, 0, sizeof(p));
    p.out = a.dx;
    if (simt) {
        if (a.dx && pl.run && pl.ok())
            pl.then(simt_product(pl, a, plain, true, p));
        if (a.dw) {
            const Plain x = plan_plain(pl, a.dtype, a.x, a.xv, a.x_inner, a.rows, a.inner);
            if (pl.run && pl.ok())
                pl.then(simt_weight_product(pl, a, x, plain));
        }
        return;
    }
    Weight w;
    Rows x;
    if (a.dx)
        w = plan_weight(pl, a);
    if (a.dw)
        x = plan_rows(pl, a.dtype, a.x, a.xv, a.x_inner, a.rows, a.inner);
    if (a.dx && pl.run && pl.ok())
        pl.then(product(pl, a, dz, w, true, p));
    if (a.dw) {
        CUtensorMap *maps = nullptr;
        if (a.ends)
            maps = static_cast<CUtensorMap *>(pl.ws.take(sizeof(CUtensorMap) * 2 * a.groups));
        const int parts = weight_parts(a);
        float *part = nullptr;
        if (parts > 1)
            part = static_cast<float *>(pl.ws.take(static_cast<size_t>(parts) * a.groups *
                                                   a.inner * a.cols * 4));
        if (pl.run && pl.ok())
            pl.then(weight_product(pl, a, x, dz, maps, parts, part));
    }
}

template <typename F>
cudaError_t sized_then_run(const PtgLinear &a, size_t *need, cudaStream_t stream, F body)
{
    Plan pl;
    begin(pl, a, false, stream);
    body(pl, a);
    *need = pl.ws.used ? pl.ws.used + kAlign : 0;     // its start may have to be moved up
    if (*need > a.workspace_bytes)
        return cudaErrorMemoryAllocation;
    if (!begin(pl, a, true, stream))
        return cudaErrorNoDevice;
    body(pl, a);
    if (pl.ok())
        ptg_record_launch(pl.kernel ? pl.kernel : "linear-bias-gradient", pl.kernel != nullptr,
                          a.dtype, pl.grid, pl.block, pl.cluster);
    return pl.err;
}

} // namespace

cudaError_t ptg_linear(const PtgLinear &a, size_t *need, cudaStream_t stream)
{
    return sized_then_run(a, need, stream, forward);
}

cudaError_t ptg_linear_backward(const PtgLinear &a, size_t *need, cudaStream_t stream)
{
    return sized_then_run(a, need, stream, backward);
}
