// The products of ragged_gemm.cuh on the CUDA cores, in float32 fused
// multiply-adds over operands of any strides:
//   out[r, f] = epilogue(sum_i A(r, i) B(i, f))
// COLS: A = x, B = w of the row's group.  INNER: A = x transposed, B = dz, i
// over the rows of one group.
//
// It serves float32 products that are too small for the split into bfloat16
// parts to pay (its passes over the operands cost more than the products),
// and 16-bit operands that would have to be laid out first.  For few rows
// the weight's bytes bound it, else the multiply-adds.  A block makes a tile of TF
// features x TR rows, four features x NR rows a thread, 32 of the inner axis
// at a time through double-buffered shared memory, the next step's loads in
// registers meanwhile.  The inner axis is split over a cluster of up to eight
// blocks when the tiles are few; partial sums are added in rank order.
#pragma once

#include "ragged_decode.cuh"

namespace ptg {

struct RaggedSimtParams {
    RaggedParams p;                     // epilogue, groups; p.inner, p.cols as there
    const void *a, *b;
    long long a_row, a_inner;           // element strides of A
    long long b_inner, b_col, b_group;  // and of B
    int split;
};

constexpr int kSimtStep = 32;           // of the inner axis at a time
constexpr int kSimtThreads = 256;

template <int TF, int TR>
constexpr int ragged_simt_smem(int groups)
{
    return (2 * kSimtStep * (TF + TR + 8) + TF * TR) * 4 + 8 * groups;
}

template <typename T, bool INNER, int TF, int TR>
__global__ void __launch_bounds__(kSimtThreads) ragged_simt_kernel(const RaggedSimtParams s)
{
    constexpr int NR = TF * TR / (4 * kSimtThreads);
    constexpr int LB = kSimtStep * TF / kSimtThreads, LA = kSimtStep * TR / kSimtThreads;
    // pitches: four more floats keep 16-byte reads aligned and spread a column's
    // writes over eight banks
    constexpr int AP = TR + 4, BP = TF + 4;
    static_assert(NR >= 2 && NR % 2 == 0 && LA >= 1, "tile too small for the block");
    extern __shared__ float simt_smem[];
    float *bs = simt_smem;                               // [2][kSimtStep][BP]
    float *as = bs + 2 * kSimtStep * BP;                 // [2][kSimtStep][AP]
    float *partial = as + 2 * kSimtStep * AP;            // [TR][TF]
    int *table = reinterpret_cast<int *>(partial + TF * TR);
    __shared__ int total_end;
    const RaggedParams &p = s.p;
    const int rank = s.split > 1 ? static_cast<int>(cluster_cta_rank()) : 0;
    const int tile = blockIdx.x / s.split;
    const int tid = threadIdx.x;
    grid_dependency_wait();
    grid_launch_dependents();

    // the tile's place
    const int ft = (p.features + TF - 1) / TF;
    const int rt = tile / ft, f0 = (tile - rt * ft) * TF;
    const int out_rows = INNER ? p.cols : p.rows;
    int group = 0, n0 = rt * TR, n_end = out_rows, k0 = 0, k_end = INNER ? p.rows : p.inner;
    int grouped_end = p.rows;
    bool live = true;
    if (p.ends) {
        fill_groups(p.ends, p.groups, p.rows, TR, table, table + p.groups, &total_end);
        const GroupTable g = {table, table + p.groups, p.groups, total_end};
        grouped_end = g.end;
        if (INNER) {
            const int per = (p.cols + TR - 1) / TR;
            group = rt / per;
            n0 = (rt - group * per) * TR;
            k0 = g.start[group];
            k_end = group_end(g, group);
        } else {
            live = rt < g.tiles[p.groups - 1];
            if (live) {
                group = find_group(g, rt);
                n0 = g.start[group] + (rt - (group > 0 ? g.tiles[group - 1] : 0)) * TR;
                n_end = group_end(g, group);
            }
        }
    }
    const int steps = live ? (k_end - k0 + kSimtStep - 1) / kSimtStep : 0;
    const int s0 = static_cast<int>(static_cast<long long>(steps) * rank / s.split);
    const int s1 = static_cast<int>(static_cast<long long>(steps) * (rank + 1) / s.split);
    const T *a = static_cast<const T *>(s.a);
    const T *b = static_cast<const T *>(s.b) + (INNER ? 0 : group * s.b_group);

    const bool b_by_col = s.b_col == 1 || s.b_inner != 1;     // which axis neighbours share
    const bool a_by_inner = s.a_inner == 1 || s.a_row != 1;
    float ra[LA], rb[LB];
    auto fetch = [&](int step) {
        const int k = k0 + step * kSimtStep;
#pragma unroll
        for (int j = 0; j < LB; j++) {
            const int e = j * kSimtThreads + tid;
            const int i = b_by_col ? e / TF : e % kSimtStep;
            const int f = b_by_col ? e % TF : e / kSimtStep;
            rb[j] = k + i < k_end && f0 + f < p.features
                        ? to_float(b[(k + i) * s.b_inner + (f0 + f) * s.b_col])
                        : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < LA; j++) {
            const int e = j * kSimtThreads + tid;
            const int i = a_by_inner ? e % kSimtStep : e / TR;
            const int r = a_by_inner ? e / kSimtStep : e % TR;
            ra[j] = k + i < k_end && n0 + r < n_end
                        ? to_float(a[(n0 + r) * s.a_row + (k + i) * s.a_inner])
                        : 0.0f;
        }
    };
    auto put = [&](int buf) {
#pragma unroll
        for (int j = 0; j < LB; j++) {
            const int e = j * kSimtThreads + tid;
            const int i = b_by_col ? e / TF : e % kSimtStep;
            const int f = b_by_col ? e % TF : e / kSimtStep;
            bs[(buf * kSimtStep + i) * BP + f] = rb[j];
        }
#pragma unroll
        for (int j = 0; j < LA; j++) {
            const int e = j * kSimtThreads + tid;
            const int i = a_by_inner ? e % kSimtStep : e / TR;
            const int r = a_by_inner ? e / kSimtStep : e % TR;
            as[(buf * kSimtStep + i) * AP + r] = ra[j];
        }
    };

    const int tx = tid % (TF / 4), ty = tid / (TF / 4);
    Float2 acc[NR][2];
#pragma unroll
    for (int r = 0; r < NR; r++)
        acc[r][0] = acc[r][1] = pair(0.0f, 0.0f);
    if (s0 < s1)
        fetch(s0);
    for (int step = s0; step < s1; step++) {
        const int buf = (step - s0) & 1;
        put(buf);
        __syncthreads();
        if (step + 1 < s1)
            fetch(step + 1);
#pragma unroll 8
        for (int i = 0; i < kSimtStep; i++) {
            const float4 q = *reinterpret_cast<const float4 *>(
                &bs[(buf * kSimtStep + i) * BP + tx * 4]);
            const Float2 q0 = pair(q.x, q.y), q1 = pair(q.z, q.w);
            float x[NR];
            const float *xs = &as[(buf * kSimtStep + i) * AP + ty * NR];
            if constexpr (NR % 4 == 0) {
#pragma unroll
                for (int r = 0; r < NR; r += 4)
                    *reinterpret_cast<float4 *>(x + r) = *reinterpret_cast<const float4 *>(xs + r);
            } else {
#pragma unroll
                for (int r = 0; r < NR; r += 2)
                    *reinterpret_cast<float2 *>(x + r) = *reinterpret_cast<const float2 *>(xs + r);
            }
#pragma unroll
            for (int r = 0; r < NR; r++) {
                const Float2 xx = pair(x[r], x[r]);
                acc[r][0] = fma2(xx, q0, acc[r][0]);
                acc[r][1] = fma2(xx, q1, acc[r][1]);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < NR; r++) {
        float4 q;
        split(acc[r][0], q.x, q.y);
        split(acc[r][1], q.z, q.w);
        *reinterpret_cast<float4 *>(&partial[(ty * NR + r) * TF + tx * 4]) = q;
    }
    if (s.split > 1)
        cluster_sync();
    else
        __syncthreads();

    if (live) {
        T *out = static_cast<T *>(p.out) + (INNER ? group * p.out_group : 0);
        T *pre = static_cast<T *>(p.pre);
        const int share = TF * TR / s.split;
        for (int e = rank * share + tid; e < (rank + 1) * share; e += kSimtThreads) {
            const int row = n0 + e / TF, feature = f0 + e % TF;
            if (row >= n_end || feature >= p.features)
                continue;
            float v;
            if (s.split > 1) {
                v = 0.0f;
                const uint32_t at = smem_addr(partial + e);
                for (int c = 0; c < s.split; c++)
                    v += ld_cluster_f32(map_to_cta(at, c));
            } else {
                v = partial[e];
            }
            const long long at = static_cast<long long>(row) * p.out_row + feature;
            if constexpr (!INNER) {
                v += load_bias<T>(p, group, feature);
                if (pre)
                    pre[at] = from_float<T>(v);
                with_activation(p.act, [&](auto act) { v = activate<act(), sizeof(T) == 2>(v); });
                if (p.residual)
                    v += to_float(static_cast<const T *>(
                        p.residual)[row * p.residual_row + feature * p.residual_inner]);
            }
            out[at] = from_float<T>(v);
        }
    }
    if (!INNER && grouped_end < p.rows)
        zero_ungrouped<T>(p, grouped_end, blockIdx.x * 8 + (tid >> 5), gridDim.x * 8);
    if (s.split > 1)
        cluster_sync();       // the others are done with this block's partial sums
}

} // namespace ptg
