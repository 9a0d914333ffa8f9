// Products over groups of rows of different lengths (a linear layer is one
// group), on CTA pairs with tcgen05.mma.cta_group::2.
//
// The weight's features are put on the M side of the tensor core and the rows
// (tokens) on the N side:
//   COLS   D[f, t] = sum_k W[g(t)][k, f] x[t, k]         forwards, and dx with W transposed
//   INNER  D[f, k] = sum_{t in group g} dz[t, f] x[t, k]  the weight's gradient
// N may be any multiple of 32 up to 256, so a group's last rows neither load,
// multiply nor store a padded tile.  It also leaves one feature per TMEM lane:
// a thread needs one bias value per tile, and a warp's 32 lanes write 32
// neighbouring features of a row.
//
// A cluster of two CTAs computes 256 features x up to 256 rows: CTA r loads
// features [128 r, 128 r + 128) and half of the rows, 64 of K at a time, into
// a ring of 128-byte-swizzled tiles.  Warps 0 and 18 issue the TMA loads of the
// two operands, warp 1 of CTA 0 the MMAs into one of two 256-column
// accumulators; warps 2 to 17 read the other one, apply bias, activation and
// residual and store.  Barriers as in gemm_tc2.cuh; every wait is bounded.  No
// TMA multicast.
//
// On B200, GPU time of short runs (the power cap makes a long one of large products
// 10-20 % slower): 8192^3 bfloat16 707-737 us = 1.49-1.56 PFLOP/s; 16384 x 2048 x 8192
// with gelu_tanh and the pre-activation stored 424 us (492-522 in a long run), with
// gelu 431-483; 64 experts, 8192 rows, 2048 x 1408 84-95 us for 370 MB of weights,
// where what a k-block costs the threads that issue loads and MMAs, and a last
// round of tiles that is mostly empty, keep it from the memory's rate.
//
// Ragged INNER axis: a k-block that crosses the end of its group must not
// meet the next group's rows (they may hold NaN, so a zero on one side is
// not enough).  Each group therefore has its own pair of tensor maps whose row
// extent ends with the group, and TMA fills zeros behind it; group_maps_kernel
// writes them from the ends on the device.
//
// CHUNKED (float32 operands, split by a pass before into three bfloat16 parts
// hi + mid + lo): every k-block runs `passes` products of parts, smallest
// first: 6 keep all terms down to 2^-24, 3 (tf32 precision mode) those down to
// 2^-16.  The tensor core truncates its accumulator at every instruction, so
// it is restarted every kChunkBlocks k-blocks and the epilogue adds the chunks
// in registers, rounding to nearest: 2.7e-7 of the result's norm from float64 at
// K = 1024.  8192 x 4096 x 4096: 1130-1160 us = 237-243 TFLOP/s, 1.42-1.46 PFLOP/s of
// MMAs.
#pragma once

#include "activation.cuh"
#include "gemm_tc2.cuh"
#include "rows.cuh"

namespace ptg {

struct RaggedParams {
    const int *ends;          // [groups] row behind each group, on the device; null: one group
    int groups, rows;
    int features;             // M side
    int cols;                 // INNER: N side
    int inner;                // COLS: K
    int a_mn;                 // COLS: the weight's features are contiguous
    int a_chunks, b_chunks;   // that map walks 64-element chunks: one load per stage
    int passes, parts;        // CHUNKED: 6 products of 3 parts per k-block, or 3 of 2
    int span;                 // rows (INNER: columns) of a tile: 256, 128 or 64
    int split;                // INNER: parts of a group's rows, each with its own result
    int act;
    uint32_t idesc;           // instruction descriptor without its N field
    void *out, *pre;
    long long out_row, out_group;       // element strides of the result
    long long out_part;                 // INNER: between the parts' results
    const void *bias;
    int bias_f32;
    const void *residual;
    long long residual_row, residual_inner;   // element strides
    int residual_small;                 // its offsets fit 32 bits
    int tma_store;                      // 16-bit results leave through maps.out and maps.pre
    const CUtensorMap *group_maps;      // INNER, several groups: a and b of each group
    int *status;
};

// A load costs the thread that issues it some 0.1 us on B200 (4096 of K: 0.35 us a
// k-block with three loads, 0.43 with four), a third of a k-block's
// MMAs at N = 256.  So a stage is two loads, by two threads: operands
// that are contiguous along features (or INNER: columns) have a map
// of dims (64, k, chunk of 64), whose one box is both of a CTA's chunks,
// where the axis is a multiple of 64; rows come in the smallest of four
// boxes that holds them.
struct RaggedMaps {
    CUtensorMap a;            // features
    CUtensorMap b;            // INNER: columns
    CUtensorMap rows[4];      // COLS: boxes of 16, 32, 64 and 128 rows
    CUtensorMap out, pre;     // results, in boxes of 32 features x kGroup rows
};

constexpr int kMaxGroups = 2048;
constexpr int kRaggedBN = 256;
// A stage is two k-blocks, or CHUNKED one k-block in all its parts, so that each
// part is loaded once for its two or three products.  Waits and commits hold up
// the thread that issues the MMAs (8192^3 bfloat16: a commit to each CTA
// per k-block 776 us, one to both 751, one for two k-blocks 724), so there is one
// of each for eight MMAs or more.
constexpr int ragged_stages(bool chunked) { return chunked ? 2 : 3; }
constexpr int kStageKb = 2;
constexpr int kMaxParts = 3;
// Sixteen epilogue warps hide each other's latencies (TMEM, residual, stores);
// CHUNKED ones keep a tile's sums in registers, 64 each.  Warps 0 and the last
// issue the loads of the two operands, warp 1 the MMAs.
constexpr int kRaggedEpiWarps = 16;
constexpr int kRaggedThreads = 32 * (3 + kRaggedEpiWarps);
constexpr int kRaggedRowWarp = 2 + kRaggedEpiWarps;
constexpr int kRaggedTile = 16384;                       // 128 rows x 64 of K, 16 bits
constexpr int kRaggedRing = 12 * kRaggedTile;
constexpr int ragged_stage_bytes(bool chunked) { return kRaggedRing / ragged_stages(chunked); }
static_assert(ragged_stage_bytes(false) == kStageKb * 2 * kRaggedTile &&
                  ragged_stage_bytes(true) == kMaxParts * 2 * kRaggedTile,
              "stages fill the ring");
constexpr int kRaggedBars = 2 * ragged_stages(false) + 4 + 1;
// the epilogue works on kGroup rows at a time: a warp's box of 32 features
constexpr int kGroup = 16;
constexpr int kRaggedBox = kGroup * 32 * 2;
constexpr int kRaggedBoxOffset = kRaggedRing;
constexpr int kRaggedBarOffset = kRaggedBoxOffset + 16 * kRaggedBox;
constexpr int kRaggedTableOffset = kRaggedBarOffset + kRaggedBars * 8 + 24;
constexpr int kRaggedSmem = kRaggedTableOffset + 2 * kMaxGroups * 4 + 1024;
static_assert(kRaggedSmem <= 232448, "shared memory budget exceeded");
constexpr int kChunkBlocks = 2;                          // k-blocks of 64 per chunk
constexpr int kFeatureBand = 8;                          // feature tiles walked per row tile

// Index in RaggedMaps::rows of the smallest box that holds n rows.
__device__ __forceinline__ int row_box(int n)
{
    return n <= 16 ? 0 : n <= 32 ? 1 : n <= 64 ? 2 : 3;
}

// Row ranges and tile counts of the groups, in shared memory.
struct GroupTable {
    int *start;      // first row
    int *tiles;      // row tiles (of `span` rows) up to and with this group
    int groups;
    int end;         // row behind the last group
};

// Fills the table: ends are taken as given, but never below the one before
// nor past the rows, so no value of theirs can lead out of the tensors.
// Called by all threads; warp 0 scans.
__device__ __forceinline__ void fill_groups(const int *ends, int groups, int rows, int span,
                                            int *start, int *tiles, int *total_end)
{
    for (int i = threadIdx.x; i < groups; i += blockDim.x)
        start[i] = ends ? min(max(__ldg(ends + i), 0), rows) : rows;
    __syncthreads();
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        int end = 0, sum = 0;
        for (int base = 0; base < groups; base += 32) {
            const int i = base + lane;
            int e = i < groups ? start[i] : 0;
            e = max(e, end);
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, e, o);
                if (lane >= o)
                    e = max(e, up);
            }
            int s = __shfl_up_sync(0xffffffffu, e, 1);
            if (lane == 0)
                s = end;
            int n = i < groups ? (e - s + span - 1) / span : 0;
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, n, o);
                if (lane >= o)
                    n += up;
            }
            n += sum;
            __syncwarp();
            if (i < groups) {
                start[i] = s;
                tiles[i] = n;
            }
            end = __shfl_sync(0xffffffffu, e, 31);
            sum = __shfl_sync(0xffffffffu, n, 31);
        }
        if (lane == 0)
            *total_end = end;
    }
    __syncthreads();
}

// Group whose tiles hold row tile t: the first with tiles[g] > t.
__device__ __forceinline__ int find_group(const GroupTable &g, int t)
{
    int lo = 0, hi = g.groups - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (g.tiles[mid] > t)
            hi = mid;
        else
            lo = mid + 1;
    }
    return lo;
}

__device__ __forceinline__ int group_end(const GroupTable &g, int i)
{
    return i + 1 < g.groups ? g.start[i + 1] : g.end;
}

// One tile of work.
struct RaggedTile {
    int group, part;
    int f0;          // first feature
    int n0, n_end;   // first row (COLS) or column (INNER), and the one behind the last
    int n;           // instruction N: a multiple of 32
    int k0;          // start of its range of the inner axis
    int k_blocks;
};

// Tile numbers are 32-bit: every role decodes each of its tiles, the ones that
// issue loads and MMAs in a single thread, where 64-bit divisions would take
// as long as some k-blocks.
template <bool INNER>
__device__ __forceinline__ unsigned ragged_tiles(const RaggedParams &p, const GroupTable &g)
{
    const unsigned ft = (p.features + 255) / 256;
    if (INNER)
        return ft * static_cast<unsigned>((p.cols + p.span - 1) / p.span) * p.groups * p.split;
    return ft * static_cast<unsigned>(g.tiles[p.groups - 1]);
}

template <bool INNER>
__device__ __forceinline__ RaggedTile ragged_tile(const RaggedParams &p, const GroupTable &g,
                                                  unsigned t)
{
    RaggedTile r;
    const unsigned ft = (p.features + 255) / 256;
    unsigned rows_t, local;
    if (INNER) {
        rows_t = (p.cols + p.span - 1) / p.span;
        const unsigned per = ft * rows_t, unit = t / per;
        local = t - unit * per;
        r.group = unit / static_cast<unsigned>(p.split);
        r.part = unit - r.group * p.split;
    } else {
        unsigned before = 0;
        r.group = 0;
        if (p.groups > 1) {
            r.group = find_group(g, static_cast<int>(t / ft));
            before = r.group > 0 ? g.tiles[r.group - 1] : 0;
        }
        rows_t = g.tiles[r.group] - before;
        local = t - before * ft;
    }
    // bands of kFeatureBand feature tiles, row tile by row tile: the clusters
    // at work at one time share their operands in L2
    const unsigned band = local / (kFeatureBand * rows_t);
    const unsigned wide = min(static_cast<unsigned>(kFeatureBand), ft - band * kFeatureBand);
    const unsigned in_band = local - band * kFeatureBand * rows_t;
    const int nt = in_band / wide;
    r.f0 = (band * kFeatureBand + in_band - nt * wide) * 256;
    const int start = g.start[r.group], end = group_end(g, r.group);
    if (INNER) {
        // whole k-blocks for each part: only the group's last one may be ragged
        const int blocks = (end - start + 63) / 64;
        const int b0 = static_cast<int>(static_cast<long long>(blocks) * r.part / p.split);
        const int b1 = static_cast<int>(static_cast<long long>(blocks) * (r.part + 1) / p.split);
        r.n0 = nt * p.span;
        r.n_end = p.cols;
        r.k0 = start + b0 * 64;
        r.k_blocks = b1 - b0;
    } else {
        r.part = 0;
        r.n0 = start + nt * p.span;
        r.n_end = end;
        r.k0 = 0;
        r.k_blocks = (p.inner + 63) / 64;
    }
    // (a map of chunks needs both CTAs' halves to be whole ones)
    const int step = INNER && p.b_chunks ? 128 : 32;
    r.n = min(p.span, (r.n_end - r.n0 + step - 1) & -step);
    return r;
}

// Parts of pass q: the smallest products first, (0,2) (1,1) (2,0) (0,1) (1,0)
// (0,0) or the last three of these; two bits per pass.
__device__ __forceinline__ void pass_parts(int passes, int q, int &pa, int &pb)
{
    const int shift = 2 * (q + 6 - passes);
    pa = (0x124 >> shift) & 3;
    pb = (0x046 >> shift) & 3;
}

// residual of rows n0 .. n0 + G - 1 (those below count) at this feature.
template <typename T, typename Offset, int G>
__device__ __forceinline__ void load_residual_at(const RaggedParams &p, int n0, int count,
                                                 int feature, T (&r)[G])
{
    const T *base = static_cast<const T *>(p.residual);
    const Offset step = static_cast<Offset>(p.residual_row);
    const Offset at = static_cast<Offset>(n0) * step +
                      static_cast<Offset>(feature) * static_cast<Offset>(p.residual_inner);
    if (count >= G) {
#pragma unroll
        for (int j = 0; j < G; j++)
            r[j] = __ldg(base + (at + j * step));
    } else {
#pragma unroll
        for (int j = 0; j < G; j++)
            if (j < count)
                r[j] = __ldg(base + (at + j * step));
    }
}

template <typename T, int G>
__device__ __forceinline__ void load_residual(const RaggedParams &p, int n0, int count,
                                              int feature, T (&r)[G])
{
    if (feature >= p.features)
        return;
    if (p.residual_small)
        load_residual_at<T, uint32_t, G>(p, n0, count, feature, r);
    else
        load_residual_at<T, long long, G>(p, n0, count, feature, r);
}

// A group's values to their place: 32 lanes write 32 neighbouring features of
// each row, through the warp's box and one TMA store (16-bit results; a lane's
// shared-memory stores have constant offsets, where global ones would cost
// address arithmetic each), or directly for the last rows of a group.
template <typename T, int G>
__device__ __forceinline__ void store_group(const RaggedParams &p, T *out, const CUtensorMap *map,
                                            uint8_t *box, int n0, int count, int f_warp,
                                            int group, const float (&v)[G])
{
    const int lane = threadIdx.x & 31;
    if constexpr (sizeof(T) == 2 && G == kGroup) {
        if (p.tma_store && count >= G) {
            if (lane == 0)
                bulk_wait_group_read<0>();       // the box's last store has read it
            __syncwarp();
            T *mine = reinterpret_cast<T *>(box) + lane;
#pragma unroll
            for (int j = 0; j < G; j++)
                mine[j * 32] = from_float<T>(v[j]);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0 && f_warp < p.features) {
                tma_store_5d(map, box, f_warp, n0, group, 0, 0);
                bulk_commit_group();
            }
            return;
        }
    }
    const int feature = f_warp + lane;
    if (feature >= p.features)
        return;
    const long long ld = p.out_row;
    out += n0 * ld + feature;
    if (count >= G) {
#pragma unroll
        for (int j = 0; j < G; j++)
            out[j * ld] = from_float<T>(v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < G; j++)
            if (j < count)
                out[j * ld] = from_float<T>(v[j]);
    }
}

// Bias, activation and residual (r, already loaded) on the values v of rows
// n0 .. and their stores.  Called by whole warps.
template <typename T, bool INNER, int G>
__device__ __forceinline__ void finish_group(const RaggedParams &p, const RaggedMaps &maps,
                                             float (&v)[G], int n0, int count, int f_warp,
                                             int group, float bias, const T (&r)[G], T *out,
                                             T *pre, uint8_t *box)
{
    constexpr bool kFast = sizeof(T) == 2;
    if (count <= 0)
        return;
    if constexpr (!INNER) {
        const Float2 b2 = pair(bias, bias);
#pragma unroll
        for (int j = 0; j < G; j += 2)
            split(add2(pair(v[j], v[j + 1]), b2), v[j], v[j + 1]);
        if (pre)
            store_group(p, pre, &maps.pre, box, n0, count, f_warp, 0, v);
        if (p.act != CUDA_MATMUL_EPILOGUE_NONE)
            with_activation(p.act, [&](auto act) {
#pragma unroll
                for (int j = 0; j < G; j++)
                    v[j] = activate<act(), kFast>(v[j]);
            });
        if (p.residual) {
#pragma unroll
            for (int j = 0; j < G; j++)
                v[j] += to_float(r[j]);
        }
    }
    store_group(p, out, &maps.out, box, n0, count, f_warp, INNER ? group : 0, v);
}

template <typename T>
__device__ __forceinline__ float load_bias(const RaggedParams &p, int group, int feature)
{
    if (!p.bias || feature >= p.features)
        return 0.0f;
    const long long i = static_cast<long long>(group) * p.features + feature;
    return p.bias_f32 ? static_cast<const float *>(p.bias)[i]
                      : to_float(static_cast<const T *>(p.bias)[i]);
}

// Rows behind the last group belong to none: their results are zero.
template <typename T>
__device__ __forceinline__ void zero_ungrouped(const RaggedParams &p, int end, int worker,
                                               int workers)
{
    for (long long r = end + static_cast<long long>(worker); r < p.rows; r += workers) {
        for (int f = threadIdx.x & 31; f < p.features; f += 32) {
            static_cast<T *>(p.out)[r * p.out_row + f] = from_float<T>(0.0f);
            if (p.pre)
                static_cast<T *>(p.pre)[r * p.out_row + f] = from_float<T>(0.0f);
        }
    }
}

// Pairs of tensor maps whose row axis (dim 1) ends with each group.
__global__ void __launch_bounds__(256)
    group_maps_kernel(const __grid_constant__ CUtensorMap a, const __grid_constant__ CUtensorMap b,
                      const int *ends, int groups, int rows, CUtensorMap *out)
{
    extern __shared__ int table[];
    __shared__ int total_end;
    grid_dependency_wait();
    grid_launch_dependents();
    fill_groups(ends, groups, rows, 64, table, table + groups, &total_end);
    const GroupTable g = {table, table + groups, groups, total_end};
    for (int i = threadIdx.x; i < 2 * groups; i += blockDim.x) {
        const int end = group_end(g, i >> 1);
        if (end == 0)
            continue;        // no rows up to here: never read
        const uint4 *src = reinterpret_cast<const uint4 *>((i & 1) ? &b : &a);
        uint4 *dst = reinterpret_cast<uint4 *>(out + i);
#pragma unroll
        for (int k = 0; k < static_cast<int>(sizeof(CUtensorMap) / 16); k++)
            dst[k] = src[k];
        tensor_map_set_dim1(out + i, end);
    }
    tensor_map_release();
}

__device__ __forceinline__ void tmem_ld_group(uint32_t taddr, uint32_t (&r)[16])
{
    tmem_ld_32x32b_x16(taddr, r);
}
__device__ __forceinline__ void tmem_ld_group(uint32_t taddr, uint32_t (&r)[8])
{
    tmem_ld_32x32b_x8(taddr, r);
}
__device__ __forceinline__ void tmem_wait_group(uint32_t (&r)[16]) { tmem_ld_wait_regs(r); }
__device__ __forceinline__ void tmem_wait_group(uint32_t (&r)[8]) { tmem_ld_wait_regs8(r); }

template <typename T, bool INNER, bool CHUNKED>
__global__ void __launch_bounds__(kRaggedThreads, 1)
    ragged_gemm_kernel(const __grid_constant__ RaggedMaps maps, const RaggedParams p)
{
    constexpr int S = ragged_stages(CHUNKED);
    constexpr int kStageBytes = ragged_stage_bytes(CHUNKED);
    // A and B of unit `sub` (k-block, or part) of a stage
    constexpr int kASub = CHUNKED ? kRaggedTile : 2 * kRaggedTile, kBSub = kASub;
    constexpr int kBOffset = CHUNKED ? kMaxParts * kRaggedTile : kRaggedTile;
    constexpr int kEpiWarps = kRaggedEpiWarps;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + kRaggedBarOffset);
    uint64_t *full = bars;
    uint64_t *empty = bars + S;
    uint64_t *tfull = bars + 2 * S;
    uint64_t *tempty = bars + 2 * S + 2;
    uint64_t *drain = bars + 2 * S + 4;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + kRaggedBars);
    volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);
    int *total_end = reinterpret_cast<int *>(tmem_slot + 2);
    int *table = reinterpret_cast<int *>(smem + kRaggedTableOffset);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_cta_rank();
    const unsigned cluster = blockIdx.x >> 1;
    const unsigned nclusters = gridDim.x >> 1;

    if (warp == 0 && lane == 0) {
        if (INNER || p.inner > 0) {
            prefetch_tensor_map(&maps.a);
            prefetch_tensor_map(INNER ? &maps.b : &maps.rows[3]);
        }
        for (int s = 0; s < S; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&tfull[i], 1);
            mbar_init(&tempty[i], 2 * kEpiWarps);
        }
        mbar_init(drain, 1);
        *abort = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, 512);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    grid_dependency_wait();
    grid_launch_dependents();
    fill_groups(p.ends, p.groups, p.rows, p.span, table, table + kMaxGroups, total_end);
    const GroupTable groups = {table, table + kMaxGroups, p.groups, *total_end};
    const unsigned tiles = ragged_tiles<INNER>(p, groups);

    if (warp == 0 || warp == kRaggedRowWarp) {
        // ------------------------------------------------------------ producers (both CTAs)
        // warp 0: the features' operand, and the barrier's expected bytes; the
        // last warp: the rows' operand
        const bool first = warp == 0;
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            uint32_t issued_mask = 0, parity_mask = 0;
            bool ok = true;
            const uint32_t full_leader = map_to_cta(smem_addr(full), 0);
            for (unsigned t = cluster; ok && t < tiles; t += nclusters) {
                const RaggedTile r = ragged_tile<INNER>(p, groups, t);
                const int half = r.n / 2;
                const int f = r.f0 + static_cast<int>(rank) * 128;
                const int n = r.n0 + static_cast<int>(rank) * half;
                const int box = INNER ? 0 : row_box(half);
                const int b_boxes = p.b_chunks ? 2 : (half + 63) / 64;
                const uint32_t bytes = kRaggedTile + (INNER ? b_boxes * 8192u : 2048u << box);
                const int units = CHUNKED ? r.k_blocks : (r.k_blocks + kStageKb - 1) / kStageKb;
                const CUtensorMap *map = first ? &maps.a : INNER ? &maps.b : &maps.rows[box];
                if (INNER && p.group_maps) {
                    map = p.group_maps + 2 * r.group + (first ? 0 : 1);
                    tensor_map_acquire(map);
                }
                for (int u = 0; u < units; u++) {
                    const int count = CHUNKED ? p.parts : min(kStageKb, r.k_blocks - u * kStageKb);
                    if (!mbar_wait(&empty[stage], phase ^ 1, abort)) {
                        record_failure(abort, p.status, DEV_TIMEOUT_PRODUCER);
                        ok = false;
                        break;
                    }
                    if (first && rank == 0)
                        mbar_arrive_expect_tx(&full[stage], count * 2 * bytes);
                    const uint32_t full0 = full_leader + stage * 8;
                    constexpr int kSubs = CHUNKED ? kMaxParts : kStageKb;
#pragma unroll
                    for (int sub = 0; sub < kSubs; sub++) {
                        if (sub >= count)
                            break;
                        const int part = CHUNKED ? sub : 0;
                        uint8_t *to = smem + stage * kStageBytes +
                                      (first ? sub * kASub : kBOffset + sub * kBSub);
                        const int k = r.k0 + (CHUNKED ? u : u * kStageKb + sub) * 64;
                        if (first) {
                            if (!INNER && !p.a_mn) {
                                tma_load_5d_pair(to, map, full0, k, f, r.group, part, 0);
                            } else if (p.a_chunks) {
                                tma_load_5d_pair(to, map, full0, 0, k, f >> 6,
                                                 INNER ? part : r.group, INNER ? 0 : part);
                            } else {
#pragma unroll
                                for (int j = 0; j < 2; j++)
                                    tma_load_5d_pair(to + j * 8192, map, full0, f + j * 64, k,
                                                     INNER ? part : r.group, INNER ? 0 : part, 0);
                            }
                        } else if (!INNER) {
                            tma_load_5d_pair(to, map, full0, k, n, part, 0, 0);
                        } else if (p.b_chunks) {
                            tma_load_5d_pair(to, map, full0, 0, k, n >> 6, part, 0);
                        } else {
                            for (int j = 0; j < b_boxes; j++)
                                tma_load_5d_pair(to + j * 8192, map, full0, n + j * 64, k, part, 0,
                                                 0);
                        }
                    }
                    issued_mask |= 1u << stage;
                    parity_mask = (parity_mask & ~(1u << stage)) | (phase << stage);
                    if (++stage == S) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
            if (first && rank == 0) {
                // CTA 0's full barriers count both CTAs' bytes of every stage
                // it posted: let them land (bounded, ignores the abort flag)
                for (int s = 0; s < S; s++) {
                    if (issued_mask & (1u << s)) {
                        int no_abort = 0;
                        mbar_wait(&full[s], (parity_mask >> s) & 1u, &no_abort);
                    }
                }
            }
            if (*abort)
                settle_after_abort();
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer (CTA 0)
        if (lane == 0 && rank == 0) {
            int stage = 0;
            uint32_t phase = 0;
            long long chunk = 0;
            bool ok = true;
            const uint32_t smem_base = smem_addr(smem);
            const bool a_mn = INNER || p.a_mn;
            // descriptors of stage 0; a step of 16 bytes adds one to them
            const uint64_t a0 = smem_desc(smem_base, a_mn ? 8192 : 16, 1024, kLayoutSw128);
            const uint64_t b0 =
                smem_desc(smem_base + kBOffset, INNER ? 8192 : 16, 1024, kLayoutSw128);
            const uint32_t a_step = (a_mn ? 16 * 128 : 32) / 16;
            constexpr uint32_t kBStep = (INNER ? 16 * 128 : 32) / 16;
            const uint32_t empty0 = smem_addr(empty);
            for (unsigned t = cluster; ok && t < tiles; t += nclusters) {
                const RaggedTile r = ragged_tile<INNER>(p, groups, t);
                const uint32_t idesc = p.idesc | (static_cast<uint32_t>(r.n >> 3) << 17);
                const int units = CHUNKED ? r.k_blocks : (r.k_blocks + kStageKb - 1) / kStageKb;
                const int per = CHUNKED ? kChunkBlocks : units;
                int left = units;
                // a tile without k-blocks still hands over one (unused) chunk
                do {
                    const int acc = static_cast<int>(chunk & 1);
                    const uint32_t acc_phase = static_cast<uint32_t>((chunk >> 1) & 1);
                    chunk++;
                    if (!mbar_wait(&tempty[acc], acc_phase ^ 1, abort)) {
                        record_failure(abort, p.status, DEV_TIMEOUT_MMA);
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * kRaggedBN);
                    const int n = min(per, left);
                    left -= n;
                    for (int i = 0; i < n; i++) {
                        if (!mbar_wait(&full[stage], phase, abort)) {
                            record_failure(abort, p.status, DEV_TIMEOUT_MMA);
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const uint64_t ad = a0 + stage * (kStageBytes / 16);
                        const uint64_t bd = b0 + stage * (kStageBytes / 16);
                        auto multiply = [&](uint64_t am, uint64_t bm, bool more) {
#pragma unroll
                            for (int k = 0; k < 4; k++)
                                umma_f16_pair(d_tmem, am + k * a_step, bm + k * kBStep, idesc,
                                              more || k != 0);
                        };
                        if constexpr (CHUNKED) {
                            for (int q = 0; q < p.passes; q++) {
                                int pa, pb;
                                pass_parts(p.passes, q, pa, pb);
                                multiply(ad + pa * (kASub / 16), bd + pb * (kBSub / 16),
                                         (i | q) != 0);
                            }
                        } else {
#pragma unroll
                            for (int sub = 0; sub < kStageKb; sub++)
                                if (i * kStageKb + sub < r.k_blocks)
                                    multiply(ad + sub * (kASub / 16), bd + sub * (kBSub / 16),
                                             (i | sub) != 0);
                        }
                        umma_commit_pair_both(empty0 + stage * 8);
                        if (++stage == S) {
                            stage = 0;
                            phase ^= 1;
                        }
                    }
                    if (!ok)
                        break;
                    umma_commit_pair_both(smem_addr(&tfull[acc]));
                } while (left > 0);
            }
            umma_commit_pair(smem_addr(drain));
            int no_abort = 0;
            mbar_wait(drain, 0, &no_abort);
        }
    } else {
        // ------------------------------------------------------------ epilogue (both CTAs)
        const int quad = warp & 3;                     // TMEM lane quadrant of this warp
        const int side = (warp - 2) >> 2;              // its kCols of the 256 columns
        uint8_t *box = smem + kRaggedBoxOffset + (warp - 2) * kRaggedBox;
        constexpr int kCols = kRaggedBN / (kEpiWarps / 4);
        long long chunk = 0;
        bool ok = true;
        for (unsigned t = cluster; ok && t < tiles; t += nclusters) {
            const RaggedTile r = ragged_tile<INNER>(p, groups, t);
            const int f_warp = r.f0 + static_cast<int>(rank) * 128 + quad * 32;
            const int feature = f_warp + lane;
            const int mine = min(max(r.n - side * kCols, 0), kCols);
            const int n0 = r.n0 + side * kCols;
            T *out = static_cast<T *>(p.out) +
                     (INNER ? r.group * p.out_group + r.part * p.out_part : 0);
            T *pre = static_cast<T *>(p.pre);
            float bias = 0.0f;
            // (the chunks' sums leave room for smaller groups only)
            constexpr int G = CHUNKED ? 8 : kGroup;
            T res[G];
            if constexpr (!INNER) {
                bias = load_bias<T>(p, r.group, feature);
                if (!CHUNKED && p.residual && mine > 0)      // in flight while the products run
                    load_residual(p, n0, r.n_end - n0, feature, res);
            }
            const int chunks =
                CHUNKED ? max(1, (r.k_blocks + kChunkBlocks - 1) / kChunkBlocks) : 1;
            float total[CHUNKED ? kCols : 1];
            if (CHUNKED) {
#pragma unroll
                for (int j = 0; j < kCols; j++)
                    total[j] = 0.0f;
            }
            for (int c = 0; c < chunks; c++) {
                const int acc = static_cast<int>(chunk & 1);
                const uint32_t acc_phase = static_cast<uint32_t>((chunk >> 1) & 1);
                chunk++;
                ok = __all_sync(0xffffffffu, mbar_wait(&tfull[acc], acc_phase, abort));
                if (!ok) {
                    if (lane == 0)
                        record_failure(abort, p.status, DEV_TIMEOUT_EPILOGUE);
                    break;
                }
                tc_fence_after();
                const uint32_t t_acc = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) +
                                       static_cast<uint32_t>(acc * kRaggedBN + side * kCols);
                if constexpr (CHUNKED) {
                    if (chunks > 1) {
#pragma unroll
                        for (int h = 0; h < kCols / 16; h++) {
                            if (h * 16 < mine) {
                                uint32_t raw[16];
                                tmem_ld_32x32b_x16(t_acc + h * 16, raw);
                                tmem_ld_wait_regs(raw);
#pragma unroll
                                for (int j = 0; j < 16; j++)
                                    total[h * 16 + j] += __uint_as_float(raw[j]);
                                if (c == chunks - 1) {
                                    // the sums take the last chunk's place
#pragma unroll
                                    for (int j = 0; j < 16; j++)
                                        raw[j] = __float_as_uint(total[h * 16 + j]);
                                    tmem_st_32x32b_x16(t_acc + h * 16, raw);
                                }
                            }
                        }
                        tmem_st_wait();
                    }
                }
                if (c == chunks - 1) {
                    uint32_t raw[G];
                    if (mine > 0) {
                        tmem_ld_group(t_acc, raw);
                        if constexpr (CHUNKED && !INNER) {   // (the sums took the registers)
                            if (p.residual)
                                load_residual(p, n0, r.n_end - n0, feature, res);
                        }
                    }
#pragma unroll 1
                    for (int h = 0; h < mine; h += G) {
                        float v[G];
                        T now[G];
                        tmem_wait_group(raw);
#pragma unroll
                        for (int j = 0; j < G; j++) {
                            v[j] = __uint_as_float(raw[j]);
                            now[j] = res[j];
                        }
                        if (r.k_blocks == 0) {       // a sum over nothing
#pragma unroll
                            for (int j = 0; j < G; j++)
                                v[j] = 0.0f;
                        }
                        if (h + G < mine) {
                            tmem_ld_group(t_acc + h + G, raw);
                            if constexpr (!INNER) {
                                if (p.residual)
                                    load_residual(p, n0 + h + G, r.n_end - (n0 + h + G),
                                                  feature, res);
                            }
                        }
                        finish_group<T, INNER>(p, maps, v, n0 + h, r.n_end - (n0 + h), f_warp,
                                               r.group, bias, now, out, pre, box);
                        __syncwarp();
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0)
                    mbar_arrive_cluster_relaxed(map_to_cta(smem_addr(&tempty[acc]), 0));
            }
        }
        if (lane == 0)
            bulk_wait_group<0>();
        __syncwarp();
        if (!INNER && groups.end < p.rows)
            zero_ungrouped<T>(p, groups.end, blockIdx.x * kEpiWarps + warp - 2,
                              gridDim.x * kEpiWarps);
    }

    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    if (warp == 1) {
        __syncwarp();
        tmem_dealloc_pair(tmem_base, 512);
    }
}

} // namespace ptg
