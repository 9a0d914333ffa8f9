// Shared by the feed-forward kernels: how a tensor is walked row by row, and
// how its elements become floats.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "internal.h"

namespace ptg {

// Element offset of row r of a view whose leading axes merged into v.n axes.
__device__ __forceinline__ long long row_offset(const RowView &v, long long r)
{
    if (v.n == 1)
        return r * v.stride[0];
    if (v.n == 2 && r < (1ll << 31)) {
        const unsigned i = static_cast<unsigned>(r), e = v.ext[1], q = i / e;
        return q * v.stride[0] + (i - q * e) * v.stride[1];
    }
    long long off = 0;
    for (int d = v.n - 1; d >= 0; d--) {
        off += (r % v.ext[d]) * v.stride[d];
        r /= v.ext[d];
    }
    return off;
}

template <typename T>
__device__ __forceinline__ float to_float(T v)
{
    if constexpr (sizeof(T) == 4)
        return v;
    else if constexpr (std::is_same<T, __half>::value)
        return __half2float(v);
    else
        return __bfloat162float(v);
}

template <typename T>
__device__ __forceinline__ T from_float(float v)
{
    if constexpr (sizeof(T) == 4)
        return v;
    else if constexpr (std::is_same<T, __half>::value)
        return __float2half_rn(v);
    else
        return __float2bfloat16_rn(v);
}

// VB bytes of T as one load or store.
template <int VB>
struct RawVec;
template <>
struct RawVec<16> {
    using type = uint4;
};
template <>
struct RawVec<8> {
    using type = uint2;
};
template <>
struct RawVec<4> {
    using type = uint32_t;
};
template <>
struct RawVec<2> {
    using type = uint16_t;
};

template <typename T, int VB>
__device__ __forceinline__ void unpack_vec(const typename RawVec<VB>::type &raw,
                                           float (&v)[VB / sizeof(T)])
{
    const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
    for (int i = 0; i < VB / static_cast<int>(sizeof(T)); i++)
        v[i] = to_float(e[i]);
}

template <typename T, int VB>
__device__ __forceinline__ typename RawVec<VB>::type pack_vec(const float (&v)[VB / sizeof(T)])
{
    typename RawVec<VB>::type raw;
    T *e = reinterpret_cast<T *>(&raw);
#pragma unroll
    for (int i = 0; i < VB / static_cast<int>(sizeof(T)); i++)
        e[i] = from_float<T>(v[i]);
    return raw;
}

// N parameters (gamma, beta, bias) from element i on, in T or in float32.
template <typename T, int N>
__device__ __forceinline__ void load_params(const void *p, int is_f32, long long i, float (&v)[N])
{
    if (is_f32) {
#pragma unroll
        for (int k = 0; k < N; k++)
            v[k] = __ldg(static_cast<const float *>(p) + i + k);
    } else {
        constexpr int VB = N * static_cast<int>(sizeof(T));
        unpack_vec<T, VB>(
            __ldg(reinterpret_cast<const typename RawVec<VB>::type *>(static_cast<const T *>(p) + i)),
            v);
    }
}

// Two floats in one 64-bit register pair, and the packed arithmetic of sm_100
// (one instruction for both, each rounded as its scalar form).
struct Float2 {
    unsigned long long v;
};

__device__ __forceinline__ Float2 pair(float lo, float hi)
{
    Float2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
    return r;
}

__device__ __forceinline__ void split(Float2 a, float &lo, float &hi)
{
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(a.v));
}

__device__ __forceinline__ Float2 add2(Float2 a, Float2 b)
{
    Float2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}

__device__ __forceinline__ Float2 mul2(Float2 a, Float2 b)
{
    Float2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}

__device__ __forceinline__ Float2 fma2(Float2 a, Float2 b, Float2 c)
{
    Float2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}

// N raw vectors of a thread as pairs, and back.
template <typename T, int VB, int N, int P>
__device__ __forceinline__ void unpack_pairs(const typename RawVec<VB>::type (&raw)[N],
                                             Float2 (&out)[P])
{
    constexpr int E = VB / sizeof(T);
    float v[2 * P];
    v[2 * P - 1] = 0.0f;             // a lone element's partner
#pragma unroll
    for (int k = 0; k < N; k++) {
        float e[E];
        unpack_vec<T, VB>(raw[k], e);
#pragma unroll
        for (int i = 0; i < E; i++)
            v[k * E + i] = e[i];
    }
#pragma unroll
    for (int k = 0; k < P; k++)
        out[k] = pair(v[2 * k], v[2 * k + 1]);
}

template <typename T, int VB, int N, int P>
__device__ __forceinline__ void pack_pairs(const Float2 (&in)[P],
                                           typename RawVec<VB>::type (&raw)[N])
{
    constexpr int E = VB / sizeof(T);
    float v[2 * P];
#pragma unroll
    for (int k = 0; k < P; k++)
        split(in[k], v[2 * k], v[2 * k + 1]);
#pragma unroll
    for (int k = 0; k < N; k++) {
        float e[E];
#pragma unroll
        for (int i = 0; i < E; i++)
            e[i] = v[k * E + i];
        raw[k] = pack_vec<T, VB>(e);
    }
}

} // namespace ptg
