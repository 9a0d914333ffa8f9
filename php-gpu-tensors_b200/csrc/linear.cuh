// The passes around the products of the linear layers: operands laid out for
// TMA, and the gradient of the epilogue.
#pragma once

#include "activation.cuh"
#include "gemm_tc.cuh"
#include "ragged_gemm.cuh"
#include "rows.cuh"

namespace ptg {

// ------------------------------------------------------------ laying out
// out[part][row][ld] from a strided source of `rows` rows and `cols` columns,
// 16 bits an element: a copy (16-bit operands whose strides or alignment TMA
// cannot describe), or the bfloat16 parts hi, mid, lo of float32 operands.
// Each thread makes eight neighbouring elements (one 16-byte store); ld is a
// multiple of 8 and columns behind `cols` are zero.  Bound by memory.
struct LayParams {
    const void *src;
    RowView rows_of;
    long long inner;        // element stride of the columns
    long long rows;
    int cols, ld;
    uint16_t *out;
    long long part;         // elements between parts
    int parts;
    int vec;                // rows can be read eight elements at a time
};

__device__ __forceinline__ void store_parts(const float (&v)[8], uint16_t *out, long long part,
                                            int parts)
{
    __nv_bfloat16 h[8], m[8], l[8];
#pragma unroll
    for (int i = 0; i < 8; i++)
        split3_bf16(v[i], h[i], m[i], l[i]);
    *reinterpret_cast<uint4 *>(out) = *reinterpret_cast<const uint4 *>(h);
    *reinterpret_cast<uint4 *>(out + part) = *reinterpret_cast<const uint4 *>(m);
    if (parts > 2)
        *reinterpret_cast<uint4 *>(out + 2 * part) = *reinterpret_cast<const uint4 *>(l);
}

// Eight elements of a row from column c on; zero from `cols` on.
template <typename T>
__device__ __forceinline__ void load8(const T *row, long long inner, int c, int cols, int vec,
                                      T (&v)[8])
{
    if (vec && c + 8 <= cols) {
        const uint4 *q = reinterpret_cast<const uint4 *>(row + c);
        uint4 *d = reinterpret_cast<uint4 *>(v);
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; i++)
            d[i] = __ldg(q + i);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            v[i] = c + i < cols ? row[(c + i) * inner] : from_float<T>(0.0f);
    }
}

// Item i of a layout: eight elements of row i / (ld / 8).
template <typename T, typename Index>
struct LayItem {
    alignas(16) T v[8];
    long long at;           // element offset of its place in the first part

    __device__ __forceinline__ void load(const LayParams &p, Index i, Index per_row)
    {
        const Index r = i / per_row;
        const int c = static_cast<int>(i - r * per_row) * 8;
        load8(static_cast<const T *>(p.src) + row_offset(p.rows_of, r), p.inner, c, p.cols, p.vec,
              v);
        at = static_cast<long long>(r) * p.ld + c;
    }
    __device__ __forceinline__ void store(const LayParams &p) const
    {
        if constexpr (sizeof(T) == 2)
            *reinterpret_cast<uint4 *>(p.out + at) = *reinterpret_cast<const uint4 *>(v);
        else
            store_parts(v, p.out + at, p.part, p.parts);
    }
};

// The next item's loads are in flight while the current one is stored.
template <typename T, typename Index>
__device__ __forceinline__ void lay_out_items(const LayParams &p, Index first, Index step)
{
    const Index per_row = static_cast<Index>(p.ld / 8);
    const Index n = static_cast<Index>(p.rows) * per_row;
    if (first >= n)
        return;
    LayItem<T, Index> now, next;
    now.load(p, first, per_row);
    for (Index i = first;; i += step) {
        const bool more = n - i > step;
        if (more)
            next.load(p, i + step, per_row);
        now.store(p);
        if (!more)
            return;
        now = next;
    }
}

// One or two layouts in a launch: blocks below `first` make a, the others b.
template <typename T>
__global__ void __launch_bounds__(256)
    lay_out_kernel(const LayParams a, const LayParams b, const int first)
{
    grid_dependency_wait();
    grid_launch_dependents();
    const bool second = static_cast<int>(blockIdx.x) >= first;
    const LayParams &p = second ? b : a;
    const unsigned block = second ? blockIdx.x - first : blockIdx.x;
    const unsigned blocks = second ? gridDim.x - first : first;
    if (p.rows * (p.ld / 8) < (1ll << 31))
        lay_out_items<T, unsigned>(p, block * 256u + threadIdx.x, blocks * 256u);
    else
        lay_out_items<T, long long>(p, block * 256ll + threadIdx.x, blocks * 256ll);
}

// A contiguous copy of a view whose rows have no single stride.
template <typename T>
__global__ void __launch_bounds__(256) copy_rows_kernel(const T *src, const RowView rows_of,
                                                        long long inner, long long rows, int cols,
                                                        T *out)
{
    grid_dependency_wait();
    grid_launch_dependents();
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < rows * cols; i += gridDim.x * 256ll) {
        const long long r = i / cols;
        out[i] = src[row_offset(rows_of, r) + (i - r * cols) * inner];
    }
}

// out[i] = the parts' float32 results at i, added in order and rounded once.
// n is a multiple of 4 elements or vec is 0.
template <typename T>
__global__ void __launch_bounds__(256) add_parts_kernel(const float *parts, int count,
                                                        long long stride, long long n, int vec,
                                                        T *out)
{
    grid_dependency_wait();
    grid_launch_dependents();
    const long long step = gridDim.x * 256ll;
    if (vec) {
        for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n / 4; i += step) {
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (int k = 0; k < count; k++) {
                const float4 q = *reinterpret_cast<const float4 *>(parts + k * stride + i * 4);
                sum.x += q.x;
                sum.y += q.y;
                sum.z += q.z;
                sum.w += q.w;
            }
            const float v[4] = {sum.x, sum.y, sum.z, sum.w};
            constexpr int VB = 4 * static_cast<int>(sizeof(T));
            reinterpret_cast<typename RawVec<VB>::type *>(out)[i] = pack_vec<T, VB>(v);
        }
    } else {
        for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += step) {
            float sum = 0.0f;
            for (int k = 0; k < count; k++)
                sum += parts[k * stride + i];
            out[i] = from_float<T>(sum);
        }
    }
}

// ------------------------------------------------------------ the epilogue's gradient
// dz = grad act'(z), rounded once to the operands' type (for the two products
// behind it: a second rounding of the size of their results'), and the bias
// gradient, the column sums of dz before that rounding, in float32.  A block
// takes 64 rows of one group and 256 columns, 8 a thread in 8 row lanes, and
// writes one partial row; group_sums_kernel adds a group's partial rows in
// order.  grad and z are read and dz written once each: 8192 x 8192 bfloat16 takes
// 83 us with gelu_tanh on B200, 103 with gelu, 66-73 with the others, 62 at the copy
// rate; the derivative's instructions (25 to 35 an element) take about as long as
// the loads.
constexpr int kSlopeRows = 64;
constexpr int kSlopeCols = 256;

// Eight values as 16 bytes of a 16-bit type (unused for float).
template <typename T>
__device__ __forceinline__ uint4 pack16(const float (&v)[8])
{
    if constexpr (sizeof(T) == 2)
        return pack_vec<T, 16>(v);
    else
        return uint4{};
}

struct SlopeParams {
    const void *grad, *pre;
    RowView gv, pv;
    long long g_inner, p_inner;
    const int *ends;
    int groups, rows, cols;
    int act;
    int g_vec, p_vec;
    void *dz;               // [rows][ld]; null when grad itself serves
    int ld;
    long long part;         // float32: parts as in lay_out_kernel
    int parts;              // 0: dz stays in float32
    float *partial;         // [row tiles][cols], or null
    int strips;             // column strips: block = row tile * strips + strip
};

// Rows r0 + lane_y + 8 k of one block, kBatch at a time: all their loads are in
// flight before the first is used (64 registers, so that four blocks share an
// SM: 64 KB of loads).
template <typename T, int ACT>
__device__ __forceinline__ void slope_rows(const SlopeParams &p, int r0, int r1, int c, int lane_y,
                                           float (&sum)[8])
{
    constexpr bool kFast = sizeof(T) == 2;
    constexpr int kBatch = sizeof(T) == 2 ? 2 : 1;
#pragma unroll 1
    for (int base = r0 + lane_y; base < r1; base += 8 * kBatch) {
        alignas(16) T g[kBatch][8], z[kBatch][8];
#pragma unroll
        for (int k = 0; k < kBatch; k++) {
            const int r = base + 8 * k;
            if (r >= r1)
                break;
            load8(static_cast<const T *>(p.grad) + row_offset(p.gv, r), p.g_inner, c, p.cols,
                  p.g_vec, g[k]);
            if constexpr (ACT != CUDA_MATMUL_EPILOGUE_NONE)
                load8(static_cast<const T *>(p.pre) + row_offset(p.pv, r), p.p_inner, c, p.cols,
                      p.p_vec, z[k]);
        }
#pragma unroll
        for (int k = 0; k < kBatch; k++) {
            const int r = base + 8 * k;
            if (r >= r1)
                break;
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                v[i] = to_float(g[k][i]);
                if constexpr (ACT != CUDA_MATMUL_EPILOGUE_NONE)
                    v[i] *= activation_slope<ACT, kFast>(to_float(z[k][i]));
            }
            if (c + 8 > p.cols) {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    v[i] = c + i < p.cols ? v[i] : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < 8; i++)
                sum[i] += v[i];
            if (p.dz) {
                uint16_t *out =
                    static_cast<uint16_t *>(p.dz) + static_cast<long long>(r) * p.ld + c;
                if (sizeof(T) == 2 && p.parts)
                    *reinterpret_cast<uint4 *>(out) = pack16<T>(v);
                else if (p.parts)
                    store_parts(v, out, p.part, p.parts);
                else {
                    float *o = static_cast<float *>(p.dz) + static_cast<long long>(r) * p.ld + c;
                    *reinterpret_cast<float4 *>(o) = make_float4(v[0], v[1], v[2], v[3]);
                    *reinterpret_cast<float4 *>(o + 4) = make_float4(v[4], v[5], v[6], v[7]);
                }
            }
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(256, 4) slope_kernel(const SlopeParams p)
{
    __shared__ float acc[8][kSlopeCols + 8];
    extern __shared__ int table[];
    __shared__ int total_end;
    grid_dependency_wait();
    grid_launch_dependents();
    const int tile = blockIdx.x / p.strips, strip = blockIdx.x - tile * p.strips;
    int r0 = tile * kSlopeRows, end = p.rows;
    if (p.ends) {
        fill_groups(p.ends, p.groups, p.rows, kSlopeRows, table, table + p.groups, &total_end);
        const GroupTable groups = {table, table + p.groups, p.groups, total_end};
        if (tile >= groups.tiles[p.groups - 1])
            return;
        const int g = find_group(groups, tile);
        r0 = groups.start[g] + (tile - (g > 0 ? groups.tiles[g - 1] : 0)) * kSlopeRows;
        end = group_end(groups, g);
    }
    if (r0 >= end)
        return;
    const int r1 = min(r0 + kSlopeRows, end);
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    const int c = strip * kSlopeCols + x * 8;
    float sum[8] = {};
    if (c < p.cols)
        with_activation(p.act, [&](auto act) { slope_rows<T, act()>(p, r0, r1, c, y, sum); });
    if (!p.partial)
        return;
#pragma unroll
    for (int i = 0; i < 8; i++)
        acc[y][x * 8 + i] = sum[i];
    __syncthreads();
    const int col = strip * kSlopeCols + threadIdx.x;
    if (col < p.cols) {
        float total = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; k++)
            total += acc[k][threadIdx.x];
        p.partial[static_cast<long long>(tile) * p.cols + col] = total;
    }
}

// out[g][c] = sum of the partial rows of group g; 32 interleaved sums joined
// by a fixed tree.  blockIdx.y = g.
__global__ void __launch_bounds__(1024) group_sums_kernel(const float *partial, const int *ends,
                                                          int groups, int rows, int cols,
                                                          float *out)
{
    __shared__ float acc[32][33];
    extern __shared__ int table[];
    __shared__ int total_end;
    grid_dependency_wait();
    grid_launch_dependents();
    const int g = blockIdx.y;
    int first = 0, behind = (rows + kSlopeRows - 1) / kSlopeRows;
    if (ends) {
        fill_groups(ends, groups, rows, kSlopeRows, table, table + groups, &total_end);
        first = g > 0 ? table[groups + g - 1] : 0;
        behind = table[groups + g];
    }
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + tx;
    float sum = 0.0f;
    if (c < cols) {
#pragma unroll 4
        for (int k = first + ty; k < behind; k += 32)
            sum += partial[static_cast<long long>(k) * cols + c];
    }
    acc[ty][tx] = sum;
    __syncthreads();
    float total = acc[tx][ty];
    for (int o = 16; o > 0; o >>= 1)
        total += __shfl_xor_sync(0xffffffffu, total, o);
    const int oc = blockIdx.x * 32 + ty;
    if (tx == 0 && oc < cols)
        out[static_cast<long long>(g) * cols + oc] = total;
}

} // namespace ptg
