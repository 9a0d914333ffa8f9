// Products over groups of rows of different lengths (a linear layer is one
// group), on CTA pairs with tcgen05.mma.cta_group::2.
//
// The weight's features are put on the M side of the tensor core and the rows
// (tokens) on the N side:
//   COLS   D[f, t] = sum_k W[g(t)][k, f] x[t, k]         forwards, and dx with W transposed
//   INNER  D[f, k] = sum_{t in group g} dz[t, f] x[t, k]  the weight's gradient
// N may be any multiple of 32 up to 256, so the last rows of a group cost an
// instruction of their own length where a 256-row M side would run (and
// throw away) a whole tile: with 64 groups of 128 rows on average a quarter of
// the work.  It also leaves one feature per TMEM lane: a thread needs
// one bias value per tile, and a warp's 32 lanes write 32 neighbouring
// features of a row.
//
// A cluster of two CTAs computes 256 features x up to 256 rows: CTA r loads
// features [128 r, 128 r + 128) and half of the rows, 64 of K at a time, into
// a 6-stage ring of 128-byte-swizzled tiles.  Warp 0 issues the TMA loads,
// warp 1 of CTA 0 the MMAs into one of two 256-column accumulators, the other
// warps read the other one, apply bias, activation and residual and store.
// Barriers as in gemm_tc2.cuh; every wait is bounded.  No TMA multicast.
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
// in registers, rounding to nearest.
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
    int passes;               // CHUNKED: products of parts per k-block, 3 or 6
    int act;
    uint32_t idesc;           // instruction descriptor without its N field
    void *out, *pre;
    long long out_row, out_group;       // element strides of the result
    const void *bias;
    int bias_f32;
    const void *residual;
    long long residual_row, residual_inner;   // element strides
    const CUtensorMap *group_maps;      // INNER, several groups: a and b of each group
    int *status;
};

struct RaggedMaps {
    CUtensorMap a;            // features
    CUtensorMap b;            // rows: a box of half a tile (COLS), or as a (INNER)
    CUtensorMap b16;          // COLS: the same in boxes of 16 rows
};

constexpr int kMaxGroups = 2048;
constexpr int kRaggedBN = 256;
constexpr int kRaggedStages = 6;
// Sixteen epilogue warps hide each other's latencies (TMEM, residual, stores);
// CHUNKED ones keep a tile's sums in registers, 64 each.
constexpr int kRaggedEpiWarps = 16;
constexpr int kRaggedThreads = 32 * (2 + kRaggedEpiWarps);
constexpr int kRaggedTile = 16384;                       // 128 rows x 64 of K, 16 bits
constexpr int kRaggedRing = kRaggedStages * 2 * kRaggedTile;
constexpr int kRaggedBars = 2 * kRaggedStages + 4 + 1;
constexpr int kRaggedTableOffset = kRaggedRing + kRaggedBars * 8 + 24;
constexpr int kRaggedSmem = kRaggedTableOffset + 2 * kMaxGroups * 4 + 1024;
static_assert(kRaggedSmem <= 232448, "shared memory budget exceeded");
constexpr int kChunkBlocks = 2;                          // k-blocks of 64 per chunk
constexpr int kFeatureBand = 8;                          // feature tiles walked per row tile

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
    int group;
    int f0;          // first feature
    int n0, n_end;   // first row (COLS) or column (INNER), and the one behind the last
    int n;           // instruction N: a multiple of 32
    int k0, k_end;   // range of the inner axis
    int k_blocks;
};

template <bool INNER>
__device__ __forceinline__ long long ragged_tiles(const RaggedParams &p, const GroupTable &g)
{
    const long long ft = (p.features + 255) / 256;
    if (INNER)
        return ft * ((p.cols + kRaggedBN - 1) / kRaggedBN) * p.groups;
    return ft * g.tiles[p.groups - 1];
}

template <bool INNER>
__device__ __forceinline__ RaggedTile ragged_tile(const RaggedParams &p, const GroupTable &g,
                                                  long long t)
{
    RaggedTile r;
    const int ft = (p.features + 255) / 256;
    int rows_t, local;
    if (INNER) {
        rows_t = (p.cols + kRaggedBN - 1) / kRaggedBN;
        const int per = ft * rows_t;
        r.group = static_cast<int>(t / per);
        local = static_cast<int>(t - static_cast<long long>(r.group) * per);
    } else {
        r.group = find_group(g, static_cast<int>(t / ft));
        const int before = r.group > 0 ? g.tiles[r.group - 1] : 0;
        rows_t = g.tiles[r.group] - before;
        local = static_cast<int>(t - static_cast<long long>(before) * ft);
    }
    // bands of kFeatureBand feature tiles, row tile by row tile: the clusters
    // at work at one time share their operands in L2
    const int band = local / (kFeatureBand * rows_t);
    const int wide = min(kFeatureBand, ft - band * kFeatureBand);
    const int in_band = local - band * kFeatureBand * rows_t;
    const int nt = in_band / wide;
    r.f0 = (band * kFeatureBand + in_band % wide) * 256;
    const int start = g.start[r.group], end = group_end(g, r.group);
    if (INNER) {
        r.n0 = nt * kRaggedBN;
        r.n_end = p.cols;
        r.k0 = start;
        r.k_end = end;
    } else {
        r.n0 = start + nt * kRaggedBN;
        r.n_end = end;
        r.k0 = 0;
        r.k_end = p.inner;
    }
    r.n = min(kRaggedBN, (r.n_end - r.n0 + 31) & ~31);
    r.k_blocks = (r.k_end - r.k0 + 63) / 64;
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

// The epilogue works on kGroup rows at a time: lane = feature, so a warp
// reads and writes 32 neighbouring features of each row.
constexpr int kGroup = 16;

// residual of rows n0 .. n0 + kGroup - 1 (those below count) at this feature.
template <typename T>
__device__ __forceinline__ void load_residual(const RaggedParams &p, int n0, int count,
                                              int feature, T (&r)[kGroup])
{
    if (feature >= p.features)
        return;
    const T *q = static_cast<const T *>(p.residual) + feature * p.residual_inner +
                 n0 * p.residual_row;
    if (count >= kGroup) {
#pragma unroll
        for (int j = 0; j < kGroup; j++)
            r[j] = __ldg(q + j * p.residual_row);
    } else {
#pragma unroll
        for (int j = 0; j < kGroup; j++)
            if (j < count)
                r[j] = __ldg(q + j * p.residual_row);
    }
}

template <typename T>
__device__ __forceinline__ void store_group(T *out, long long ld, int count,
                                            const float (&v)[kGroup])
{
    if (count >= kGroup) {
#pragma unroll
        for (int j = 0; j < kGroup; j++)
            out[j * ld] = from_float<T>(v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < kGroup; j++)
            if (j < count)
                out[j * ld] = from_float<T>(v[j]);
    }
}

// Bias, activation and residual (r, already loaded) on the values v of rows
// n0 .. and their stores.
template <typename T, bool INNER>
__device__ __forceinline__ void finish_group(const RaggedParams &p, float (&v)[kGroup], int n0,
                                             int count, int feature, float bias,
                                             const T (&r)[kGroup], T *out, T *pre)
{
    constexpr bool kFast = sizeof(T) == 2;
    if (feature >= p.features || count <= 0)
        return;
    const long long ld = p.out_row;
    if constexpr (!INNER) {
#pragma unroll
        for (int j = 0; j < kGroup; j++)
            v[j] += bias;
        if (pre)
            store_group(pre + n0 * ld + feature, ld, count, v);
        if (p.act != CUDA_MATMUL_EPILOGUE_NONE)
            with_activation(p.act, [&](auto act) {
#pragma unroll
                for (int j = 0; j < kGroup; j++)
                    v[j] = activate<act(), kFast>(v[j]);
            });
        if (p.residual) {
#pragma unroll
            for (int j = 0; j < kGroup; j++)
                v[j] += to_float(r[j]);
        }
    }
    store_group(out + n0 * ld + feature, ld, count, v);
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

template <typename T, bool INNER, bool CHUNKED>
__global__ void __launch_bounds__(kRaggedThreads, 1)
    ragged_gemm_kernel(const __grid_constant__ RaggedMaps maps, const RaggedParams p)
{
    constexpr int S = kRaggedStages;
    constexpr int kEpiWarps = kRaggedEpiWarps;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + kRaggedRing);
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
    const long long cluster = blockIdx.x >> 1;
    const long long nclusters = gridDim.x >> 1;

    if (warp == 0 && lane == 0) {
        if (INNER || p.inner > 0) {
            prefetch_tensor_map(&maps.a);
            prefetch_tensor_map(&maps.b);
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
    fill_groups(p.ends, p.groups, p.rows, kRaggedBN, table, table + kMaxGroups, total_end);
    const GroupTable groups = {table, table + kMaxGroups, p.groups, *total_end};
    const long long tiles = ragged_tiles<INNER>(p, groups);
    const int passes = CHUNKED ? p.passes : 1;

    if (warp == 0) {
        // ------------------------------------------------------------ producer (both CTAs)
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            uint32_t issued_mask = 0, parity_mask = 0;
            bool ok = true;
            for (long long t = cluster; ok && t < tiles; t += nclusters) {
                const RaggedTile r = ragged_tile<INNER>(p, groups, t);
                const int half = r.n / 2;
                const int f = r.f0 + static_cast<int>(rank) * 128;
                const int n = r.n0 + static_cast<int>(rank) * half;
                const int b_boxes = INNER ? (half + 63) / 64 : half == 128 ? 1 : half / 16;
                const uint32_t bytes =
                    kRaggedTile + (INNER ? b_boxes * 8192u : static_cast<uint32_t>(half) * 128u);
                const int iters = r.k_blocks * passes;
                const CUtensorMap *map_a = &maps.a, *map_b = &maps.b;
                if (INNER && p.group_maps) {
                    map_a = p.group_maps + 2 * r.group;
                    map_b = map_a + 1;
                    tensor_map_acquire(map_a);
                    tensor_map_acquire(map_b);
                }
                for (int i = 0; i < iters; i++) {
                    int pa = 0, pb = 0, kb = i;
                    if (CHUNKED) {
                        kb = i / passes;
                        pass_parts(passes, i - kb * passes, pa, pb);
                    }
                    if (!mbar_wait(&empty[stage], phase ^ 1, abort)) {
                        record_failure(abort, p.status, DEV_TIMEOUT_PRODUCER);
                        ok = false;
                        break;
                    }
                    uint8_t *sa = smem + stage * 2 * kRaggedTile;
                    uint8_t *sb = sa + kRaggedTile;
                    if (rank == 0)
                        mbar_arrive_expect_tx(&full[stage], 2 * bytes);
                    const uint32_t full0 = map_to_cta(smem_addr(&full[stage]), 0);
                    const int k = r.k0 + kb * 64;
                    if (INNER) {
#pragma unroll
                        for (int j = 0; j < 2; j++)
                            tma_load_5d_pair(sa + j * 8192, map_a, full0, f + j * 64, k, pa, 0, 0);
                        for (int j = 0; j < b_boxes; j++)
                            tma_load_5d_pair(sb + j * 8192, map_b, full0, n + j * 64, k, pb, 0, 0);
                    } else {
                        if (p.a_mn) {
#pragma unroll
                            for (int j = 0; j < 2; j++)
                                tma_load_5d_pair(sa + j * 8192, &maps.a, full0, f + j * 64, k,
                                                 r.group, pa, 0);
                        } else {
                            tma_load_5d_pair(sa, &maps.a, full0, k, f, r.group, pa, 0);
                        }
                        if (half == 128) {
                            tma_load_5d_pair(sb, &maps.b, full0, k, n, pb, 0, 0);
                        } else {
                            for (int j = 0; j < b_boxes; j++)
                                tma_load_5d_pair(sb + j * 2048, &maps.b16, full0, k, n + j * 16,
                                                 pb, 0, 0);
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
            if (rank == 0) {
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
            const uint32_t a_lbo = a_mn ? 8192 : 16, a_step = a_mn ? 16 * 128 : 32;
            const uint32_t b_lbo = INNER ? 8192 : 16, b_step = INNER ? 16 * 128 : 32;
            for (long long t = cluster; ok && t < tiles; t += nclusters) {
                const RaggedTile r = ragged_tile<INNER>(p, groups, t);
                const uint32_t idesc = p.idesc | (static_cast<uint32_t>(r.n >> 3) << 17);
                const int per = CHUNKED ? kChunkBlocks * passes : r.k_blocks;
                int left = r.k_blocks * passes;
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
                        const uint32_t sa = smem_base + stage * 2 * kRaggedTile;
                        const uint32_t sb = sa + kRaggedTile;
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const uint64_t ad =
                                smem_desc(sa + k * a_step, a_lbo, 1024, kLayoutSw128);
                            const uint64_t bd =
                                smem_desc(sb + k * b_step, b_lbo, 1024, kLayoutSw128);
                            umma_f16_pair(d_tmem, ad, bd, idesc, (i | k) != 0);
                        }
                        const uint32_t e0 = smem_addr(&empty[stage]);
                        umma_commit_pair(e0);
                        umma_commit_pair(map_to_cta(e0, 1));
                        if (++stage == S) {
                            stage = 0;
                            phase ^= 1;
                        }
                    }
                    if (!ok)
                        break;
                    const uint32_t f0 = smem_addr(&tfull[acc]);
                    umma_commit_pair(f0);
                    umma_commit_pair(map_to_cta(f0, 1));
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
        constexpr int kCols = kRaggedBN / (kEpiWarps / 4);
        long long chunk = 0;
        bool ok = true;
        for (long long t = cluster; ok && t < tiles; t += nclusters) {
            const RaggedTile r = ragged_tile<INNER>(p, groups, t);
            const int feature = r.f0 + static_cast<int>(rank) * 128 + quad * 32 + lane;
            const int mine = min(max(r.n - side * kCols, 0), kCols);   // multiple of 32
            const int n0 = r.n0 + side * kCols;
            T *out = static_cast<T *>(p.out) + (INNER ? r.group * p.out_group : 0);
            T *pre = static_cast<T *>(p.pre);
            float bias = 0.0f;
            T res[kGroup];
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
                    uint32_t raw[kGroup];
                    if (mine > 0) {
                        tmem_ld_32x32b_x16(t_acc, raw);
                        if constexpr (CHUNKED && !INNER) {   // (the sums took the registers)
                            if (p.residual)
                                load_residual(p, n0, r.n_end - n0, feature, res);
                        }
                    }
#pragma unroll 1
                    for (int h = 0; h < mine; h += kGroup) {
                        float v[kGroup];
                        T now[kGroup];
                        tmem_ld_wait_regs(raw);
#pragma unroll
                        for (int j = 0; j < kGroup; j++) {
                            v[j] = r.k_blocks > 0 ? __uint_as_float(raw[j]) : 0.0f;
                            now[j] = res[j];
                        }
                        if (h + kGroup < mine) {
                            tmem_ld_32x32b_x16(t_acc + h + kGroup, raw);
                            if constexpr (!INNER) {
                                if (p.residual)
                                    load_residual(p, n0 + h + kGroup, r.n_end - (n0 + h + kGroup),
                                                  feature, res);
                            }
                        }
                        finish_group<T, INNER>(p, v, n0 + h, r.n_end - (n0 + h), feature, bias, now,
                                               out, pre);
                        __syncwarp();
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0)
                    mbar_arrive_cluster(map_to_cta(smem_addr(&tempty[acc]), 0));
            }
        }
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
