// The products of ragged_gemm.cuh on the CUDA cores, in float32 fused
// multiply-adds over operands of any strides:
//   out[r, f] = epilogue(sum_i A(r, i) B(i, f))
// COLS: A = x, B = w of the row's group.  INNER: A = x transposed, B = dz, i
// over the rows of one group.
//
// It serves float32 products that are too small for the split into bfloat16
// parts to pay (its passes over the operands cost more than the products),
// 16-bit operands that would have to be laid out first, and the gradients of
// a few rows, whose dz stays in float32 (TZ): so few roundings to 16 bits
// would not average out in the products.  For few rows
// the weight's bytes bound it, else the multiply-adds.  A block makes a tile of TF
// features x TR rows, four features x NR rows a thread, 32 of the inner axis
// at a time through double-buffered shared memory, the next step's loads in
// registers meanwhile.  The inner axis is split over a cluster of up to eight
// blocks when the tiles are few; partial sums are added in rank order.  On B200:
// 8 x 4096 x 4096 float32 37 us (67 MB), 512 x 1024 x 1024 50 us, 4096 x 1024 x 1024
// 290 us = 30 TFLOP/s (128 x 64 tiles, with 174 registers, were no faster).
#pragma once

#include "ragged_decode.cuh"

namespace ptg {

struct RaggedSimtParams {
    RaggedParams p;                     // epilogue, groups; p.inner, p.cols as there
    const void *a, *b;
    long long a_row, a_inner;           // element strides of A
    long long b_inner, b_col, b_group;  // and of B
    int split;
    int out_f32;                        // INNER: the result is float32 whatever T is
};

constexpr int kSimtStep = 32;           // of the inner axis at a time
constexpr int kSimtThreads = 256;

template <int TF, int TR>
constexpr int ragged_simt_smem(int groups)
{
    return (2 * kSimtStep * (TF + TR + 8) + TF * TR) * 4 + 8 * groups;
}

template <typename T, typename TZ, bool INNER, int TF, int TR>
__global__ void __launch_bounds__(kSimtThreads) ragged_simt_kernel(const RaggedSimtParams s)
{
    constexpr int NR = TF * TR / (4 * kSimtThreads);
    constexpr int LB = kSimtStep * TF / kSimtThreads, LA = kSimtStep * TR / kSimtThreads;
    // pitches: four more floats keep 16-byte reads aligned and spread a column's
    // writes over eight banks
    constexpr int AP = TR + 4, BP = TF + 4;
    using TA = std::conditional_t<INNER, T, TZ>;
    using TB = std::conditional_t<INNER, TZ, T>;
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
    const TA *a = static_cast<const TA *>(s.a);
    const TB *b = static_cast<const TB *>(s.b) + (INNER ? 0 : group * s.b_group);

    // Neighbouring threads read along the axis that is contiguous; every load of
    // a thread then differs from its first by a fixed step, and its place on
    // the other axis by a fixed count.
    const bool b_by_col = s.b_col == 1 || s.b_inner != 1;
    const bool a_by_inner = s.a_inner == 1 || s.a_row != 1;
    const int bi = b_by_col ? tid / TF : tid % kSimtStep;
    const int bf = b_by_col ? tid % TF : tid / kSimtStep;
    const int bi_step = b_by_col ? kSimtThreads / TF : 0;
    const int bf_step = b_by_col ? 0 : kSimtThreads / kSimtStep;
    const int ai = a_by_inner ? tid % kSimtStep : tid / TR;
    const int ar = a_by_inner ? tid / kSimtStep : tid % TR;
    const int ai_step = a_by_inner ? 0 : kSimtThreads / TR;
    const int ar_step = a_by_inner ? kSimtThreads / kSimtStep : 0;
    const long long b_step = bi_step * s.b_inner + bf_step * s.b_col;
    const long long a_step = ai_step * s.a_inner + ar_step * s.a_row;
    const long long first = k0 + static_cast<long long>(s0) * kSimtStep;
    const TB *b_at = b + (first + bi) * s.b_inner + (f0 + bf) * s.b_col;
    const TA *a_at = a + (n0 + ar) * s.a_row + (first + ai) * s.a_inner;
    float ra[2][LA], rb[2][LB];
    // the next step's elements into register set `set`; steps come in order
    auto fetch = [&](int set, int step) {
        const int left = k_end - (k0 + step * kSimtStep);
#pragma unroll
        for (int j = 0; j < LB; j++)
            rb[set][j] = bi + j * bi_step < left && f0 + bf + j * bf_step < p.features
                             ? to_float(b_at[j * b_step])
                             : 0.0f;
#pragma unroll
        for (int j = 0; j < LA; j++)
            ra[set][j] = ai + j * ai_step < left && n0 + ar + j * ar_step < n_end
                             ? to_float(a_at[j * a_step])
                             : 0.0f;
        b_at += kSimtStep * s.b_inner;
        a_at += kSimtStep * s.a_inner;
    };
    const int b_put = bi * BP + bf, b_put_step = bi_step * BP + bf_step;
    const int a_put = ai * AP + ar, a_put_step = ai_step * AP + ar_step;
    auto put = [&](int set) {
#pragma unroll
        for (int j = 0; j < LB; j++)
            bs[set * kSimtStep * BP + b_put + j * b_put_step] = rb[set][j];
#pragma unroll
        for (int j = 0; j < LA; j++)
            as[set * kSimtStep * AP + a_put + j * a_put_step] = ra[set][j];
    };

    const int tx = tid % (TF / 4), ty = tid / (TF / 4);
    Float2 acc[NR][2];
#pragma unroll
    for (int r = 0; r < NR; r++)
        acc[r][0] = acc[r][1] = pair(0.0f, 0.0f);
#pragma unroll
    for (int set = 0; set < 2; set++)
        if (s0 + set < s1)
            fetch(set, s0 + set);
    for (int base = s0; base < s1; base += 2) {
#pragma unroll
        for (int set = 0; set < 2; set++) {
            if (base + set >= s1)
                break;
            put(set);
            __syncthreads();
            if (base + set + 2 < s1)
                fetch(set, base + set + 2);
#pragma unroll 8
            for (int i = 0; i < kSimtStep; i++) {
                const float4 q = *reinterpret_cast<const float4 *>(
                    &bs[(set * kSimtStep + i) * BP + tx * 4]);
                const Float2 q0 = pair(q.x, q.y), q1 = pair(q.z, q.w);
                float x[NR];
                const float *xs = &as[(set * kSimtStep + i) * AP + ty * NR];
                if constexpr (NR % 4 == 0) {
#pragma unroll
                    for (int r = 0; r < NR; r += 4)
                        *reinterpret_cast<float4 *>(x + r) =
                            *reinterpret_cast<const float4 *>(xs + r);
                } else {
#pragma unroll
                    for (int r = 0; r < NR; r += 2)
                        *reinterpret_cast<float2 *>(x + r) =
                            *reinterpret_cast<const float2 *>(xs + r);
                }
#pragma unroll
                for (int r = 0; r < NR; r++) {
                    const Float2 xx = pair(x[r], x[r]);
                    acc[r][0] = fma2(xx, q0, acc[r][0]);
                    acc[r][1] = fma2(xx, q1, acc[r][1]);
                }
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
            if constexpr (INNER && sizeof(T) == 2) {
                if (s.out_f32) {
                    static_cast<float *>(p.out)[group * p.out_group + at] = v;
                    continue;
                }
            }
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
