// The products of ragged_gemm.cuh (COLS) for few rows, where reading the
// weight is the work: a step of decoding, or a handful of rows per expert.
//
// One CTA takes 128 features x up to 64 rows (features on the M side as there:
// the weight streams through the M side at full width while N is only as long
// as the rows, a multiple of 16).  The inner axis is split over a cluster of
// up to eight CTAs, so that a 4096 x 4096 weight, which has only 32 feature
// tiles, is read by 256 CTAs; each writes its partial sums to its own
// shared memory and takes a share of the rows, adding the partial sums of all
// CTAs in rank order (the result does not depend on timing) and finishing
// them.  96 KB of tiles in flight per CTA and two CTAs per SM keep
// enough loads outstanding for the memory's latency: 8 x 4096 x 4096 bfloat16 takes
// 10.4 us in a run of calls on weights that come from memory (8.5 where L2 has
// them; alone, with its launch, 14), the weight's 34 MB 5.1 at the copy rate; the
// pair kernel's 16 tiles take 21.
#pragma once

#include "ragged_gemm.cuh"

namespace ptg {

constexpr int kDecodeRows = 64;
constexpr int kDecodeStages = 4;
constexpr int kDecodeThreads = 192;
constexpr int kDecodeATile = 16384;
constexpr int kDecodeStage = kDecodeATile + kDecodeRows * 128;
constexpr int kDecodeRing = kDecodeStages * kDecodeStage;
constexpr int kDecodeBars = 2 * kDecodeStages + 1;
constexpr int kDecodeTable = kDecodeRing + kDecodeBars * 8 + 24;
static_assert(kDecodeRows * 128 * 4 <= kDecodeRing, "partial sums fit in the ring");

// Shared memory for `groups` groups (no table without ends).
constexpr int decode_smem(int groups) { return kDecodeTable + 8 * groups + 1024; }

__device__ __forceinline__ float ld_cluster_f32(uint32_t cluster_addr)
{
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr) : "memory");
    return v;
}

template <typename T>
__global__ void __launch_bounds__(kDecodeThreads)
    ragged_decode_kernel(const __grid_constant__ RaggedMaps maps, const RaggedParams p,
                         const int split)
{
    constexpr int S = kDecodeStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + kDecodeRing);
    uint64_t *empty = full + S;
    uint64_t *done = full + 2 * S;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(full + kDecodeBars);
    volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);
    int *total_end = reinterpret_cast<int *>(tmem_slot + 2);
    int *table = reinterpret_cast<int *>(smem + kDecodeTable);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int rank = split > 1 ? static_cast<int>(cluster_cta_rank()) : 0;
    const int tile = blockIdx.x / split;

    if (threadIdx.x == 0) {
        if (p.inner > 0) {
            prefetch_tensor_map(&maps.a);
            prefetch_tensor_map(&maps.rows[0]);
        }
        for (int s = 0; s < S; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(done, 1);
        *abort = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 64);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    grid_dependency_wait();
    grid_launch_dependents();

    // which tile: feature tiles of one row tile are neighbours
    const int ft = (p.features + 127) / 128;
    const int rt = tile / ft, f0 = (tile - rt * ft) * 128;
    int group = 0, n0 = rt * kDecodeRows, n_end = p.rows, grouped_end = p.rows;
    bool live = n0 < p.rows;
    if (p.ends) {
        fill_groups(p.ends, p.groups, p.rows, kDecodeRows, table, table + p.groups, total_end);
        const GroupTable g = {table, table + p.groups, p.groups, *total_end};
        grouped_end = g.end;
        live = rt < g.tiles[p.groups - 1];
        if (live) {
            group = find_group(g, rt);
            n0 = g.start[group] + (rt - (group > 0 ? g.tiles[group - 1] : 0)) * kDecodeRows;
            n_end = group_end(g, group);
        }
    }
    const int rows = live ? min(kDecodeRows, n_end - n0) : 0;
    const int n = (rows + 15) & ~15;
    const int box = row_box(n);
    const int blocks = (p.inner + 63) / 64;
    const int kb0 = static_cast<int>(static_cast<long long>(blocks) * rank / split);
    const int kb1 = live ? static_cast<int>(static_cast<long long>(blocks) * (rank + 1) / split)
                         : kb0;

    if (warp == 0 && lane == 0) {
        // ------------------------------------------------------------ loads
        uint32_t phase = 0;
        int stage = 0, issued = 0;
        for (int kb = kb0; kb < kb1; kb++) {
            if (!mbar_wait(&empty[stage], phase ^ 1, abort)) {
                record_failure(abort, p.status, DEV_TIMEOUT_PRODUCER);
                break;
            }
            uint8_t *sa = smem + stage * kDecodeStage;
            uint8_t *sb = sa + kDecodeATile;
            mbar_arrive_expect_tx(&full[stage], kDecodeATile + (2048 << box));
            const int k = kb * 64;
            if (!p.a_mn) {
                tma_load_5d(sa, &maps.a, &full[stage], k, f0, group, 0, 0);
            } else if (p.a_chunks) {
                tma_load_5d(sa, &maps.a, &full[stage], 0, k, f0 >> 6, group, 0);
            } else {
#pragma unroll
                for (int j = 0; j < 2; j++)
                    tma_load_5d(sa + j * 8192, &maps.a, &full[stage], f0 + j * 64, k, group, 0, 0);
            }
            tma_load_5d(sb, &maps.rows[box], &full[stage], k, n0, 0, 0, 0);
            issued++;
            if (++stage == S) {
                stage = 0;
                phase ^= 1;
            }
        }
        // every load must have landed before the ring is reused or freed
        // (bounded, ignores the abort flag)
        for (int i = max(0, issued - S); i < issued; i++) {
            int no_abort = 0;
            mbar_wait(&full[i % S], static_cast<uint32_t>(i / S) & 1u, &no_abort);
        }
    } else if (warp == 1 && lane == 0) {
        // ------------------------------------------------------------ MMAs
        uint32_t phase = 0;
        int stage = 0;
        const uint32_t base = smem_addr(smem);
        const uint32_t idesc = p.idesc | (static_cast<uint32_t>(n >> 3) << 17);
        const uint32_t a_lbo = p.a_mn ? 8192 : 16, a_step = p.a_mn ? 16 * 128 : 32;
        for (int kb = kb0; kb < kb1; kb++) {
            if (!mbar_wait(&full[stage], phase, abort)) {
                record_failure(abort, p.status, DEV_TIMEOUT_MMA);
                break;
            }
            tc_fence_after();
            const uint32_t sa = base + stage * kDecodeStage, sb = sa + kDecodeATile;
#pragma unroll
            for (int k = 0; k < 4; k++)
                umma_f16(tmem, smem_desc(sa + k * a_step, a_lbo, 1024, kLayoutSw128),
                         smem_desc(sb + k * 32, 16, 1024, kLayoutSw128), idesc,
                         (kb != kb0 || k != 0) ? 1u : 0u);
            umma_commit(&empty[stage]);
            if (++stage == S) {
                stage = 0;
                phase ^= 1;
            }
        }
        umma_commit(done);
        int no_abort = 0;
        mbar_wait(done, 0, &no_abort);
    }
    __syncthreads();          // products done, all loads landed: the ring is free

    // -------------------------------------------------------------- finish
    const int quad = warp & 3;
    const bool finisher = warp >= 2;
    const int f_local = quad * 32 + lane, feature = f0 + f_local;
    const uint32_t t_acc = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    float *partial = reinterpret_cast<float *>(smem);       // [row][128]
    if (split > 1) {
        if (finisher) {
            tc_fence_after();
            for (int h = 0; h < n; h += 16) {
                uint32_t raw[16];
                tmem_ld_32x32b_x16(t_acc + h, raw);
                tmem_ld_wait_regs(raw);
#pragma unroll
                for (int j = 0; j < 16; j++)
                    partial[(h + j) * 128 + f_local] = kb1 > kb0 ? __uint_as_float(raw[j]) : 0.0f;
            }
        }
        cluster_sync();
    }
    if (finisher && live) {
        const float bias = load_bias<T>(p, group, feature);
        T *out = static_cast<T *>(p.out), *pre = static_cast<T *>(p.pre);
        auto finish = [&](float v, int row) {
            if (feature >= p.features)
                return;
            const long long at = static_cast<long long>(n0 + row) * p.out_row + feature;
            v += bias;
            if (pre)
                pre[at] = from_float<T>(v);
            with_activation(p.act, [&](auto act) { v = activate<act(), sizeof(T) == 2>(v); });
            if (p.residual)
                v += to_float(static_cast<const T *>(
                    p.residual)[(n0 + row) * p.residual_row + feature * p.residual_inner]);
            out[at] = from_float<T>(v);
        };
        if (split > 1) {
            for (int row = rank; row < rows; row += split) {
                const uint32_t at = smem_addr(partial + row * 128 + f_local);
                float v = 0.0f;
                for (int c = 0; c < split; c++)
                    v += ld_cluster_f32(map_to_cta(at, c));
                finish(v, row);
            }
        } else {
            tc_fence_after();
            for (int h = 0; h < n; h += 16) {
                uint32_t raw[16];
                tmem_ld_32x32b_x16(t_acc + h, raw);
                tmem_ld_wait_regs(raw);
#pragma unroll
                for (int j = 0; j < 16; j++)
                    if (h + j < rows)
                        finish(kb1 > kb0 ? __uint_as_float(raw[j]) : 0.0f, h + j);
                __syncwarp();
            }
        }
    }
    if (finisher && grouped_end < p.rows)
        zero_ungrouped<T>(p, grouped_end, blockIdx.x * 4 + warp - 2, gridDim.x * 4);
    tc_fence_before();
    if (split > 1)
        cluster_sync();       // the others are done with this CTA's partial sums
    else
        __syncthreads();
    tc_fence_after();
    if (warp == 1) {
        __syncwarp();
        tmem_dealloc(tmem, 64);
    }
}

} // namespace ptg
