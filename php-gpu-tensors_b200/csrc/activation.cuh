// Activations of the feed-forward layers and their derivatives, in float32.
//
//   relu z+            tanh            sigmoid s(z) = 1 / (1 + e^-z)
//   silu z s(z)        gelu z P(z)     gelu_tanh z s(2 u), u = c (z + 0.044715 z^3)
//
// with P the normal distribution function and c = sqrt(2 / pi);
// (1 + tanh u) / 2 = s(2 u) turns the usual form of gelu_tanh into one
// exponential and one division.  P is taken from its tail, P(-|z|), which keeps
// its digits where 1 + erf cancels: erfcf for float32 results.  FAST serves
// results of 16 bits: the hardware's exponential and division (their errors
// and those of the arguments: |x| + 4 units of 2^-23 for e^x), and
//   P(-a) = e^(-a^2 / 2) R(a),  R(a) = t (c0 + c1 t + ... + c7 t^7),  t = 1 / (1 + 0.4 a)
// in the form of 7.1.26 in Abramowitz and Stegun's handbook, whose
// coefficients bound erf's absolute error.  These keep P within 1.6e-8, since
// dbias sums slopes in float32, and within 1e-6 of itself on [0, 14.5], where
// z P(z) leaves bfloat16's range; the exponential is the density's.
#pragma once

#include "gemm_sm100.h"

namespace ptg {

template <bool FAST>
__device__ __forceinline__ float exp_of(float x)
{
    return FAST ? __expf(x) : expf(x);
}

template <bool FAST>
__device__ __forceinline__ float divide(float a, float b)
{
    return FAST ? __fdividef(a, b) : a / b;
}

constexpr float kGeluC = 0.7978845608028654f;     // sqrt(2 / pi)
constexpr float kGeluA = 0.044715f;
constexpr float kSqrtHalf = 0.7071067811865476f;

// P(z), and e^(-z^2 / 2) for the density.
template <bool FAST>
__device__ __forceinline__ float normal_cdf(float z, float &gauss)
{
    gauss = exp_of<FAST>(-0.5f * z * z);
    if constexpr (FAST) {
        const float t = __fdividef(1.0f, fmaf(0.4f, fabsf(z), 1.0f));
        float q = fmaf(-0.0350036f, t, 0.17938237f);
        q = fmaf(q, t, -0.33261806f);
        q = fmaf(q, t, 0.20771052f);
        q = fmaf(q, t, 0.014565778f);
        q = fmaf(q, t, 0.14832395f);
        q = fmaf(q, t, 0.15799007f);
        q = fmaf(q, t, 0.15964898f);
        const float tail = q * t * gauss;             // P(-|z|)
        return z > 0.0f ? 1.0f - tail : tail;
    } else {
        return 0.5f * erfcf(-z * kSqrtHalf);
    }
}

template <int ACT, bool FAST>
__device__ __forceinline__ float activate(float z)
{
    if constexpr (ACT == CUDA_MATMUL_EPILOGUE_RELU)
        return z > 0.0f ? z : 0.0f;
    else if constexpr (ACT == CUDA_MATMUL_EPILOGUE_TANH)
        return tanhf(z);
    else if constexpr (ACT == CUDA_MATMUL_EPILOGUE_SIGMOID)
        return divide<FAST>(1.0f, 1.0f + exp_of<FAST>(-z));
    else if constexpr (ACT == CUDA_MATMUL_EPILOGUE_SILU)
        return divide<FAST>(z, 1.0f + exp_of<FAST>(-z));
    else if constexpr (ACT == CUDA_MATMUL_EPILOGUE_GELU)
    {
        float gauss;
        return z * normal_cdf<FAST>(z, gauss);
    } else if constexpr (ACT == CUDA_MATMUL_EPILOGUE_GELU_TANH) {
        const float u = kGeluC * fmaf(kGeluA * z * z, z, z);
        return divide<FAST>(z, 1.0f + exp_of<FAST>(-2.0f * u));
    } else
        return z;
}

template <int ACT, bool FAST>
__device__ __forceinline__ float activation_slope(float z)
{
    if constexpr (ACT == CUDA_MATMUL_EPILOGUE_RELU)
        return z > 0.0f ? 1.0f : 0.0f;
    else if constexpr (ACT == CUDA_MATMUL_EPILOGUE_TANH || ACT == CUDA_MATMUL_EPILOGUE_SIGMOID) {
        // even functions of z, from the exponential that is at most one: 1 - tanh^2
        // = 4 e / (1 + e)^2 with e = e^(-2 |z|), and s (1 - s) = e / (1 + e)^2 with
        // e^(-|z|); the differences would cancel in the tails, and (1 + e)^2 as
        // 1 + e (2 + e) rounds about once
        constexpr bool kTanh = ACT == CUDA_MATMUL_EPILOGUE_TANH;
        const float e = exp_of<FAST>(fabsf(z) * (kTanh ? -2.0f : -1.0f));
        return divide<FAST>(kTanh ? 4.0f * e : e, fmaf(e, 2.0f + e, 1.0f));
    } else if constexpr (ACT == CUDA_MATMUL_EPILOGUE_SILU) {
        const float s = divide<FAST>(1.0f, 1.0f + exp_of<FAST>(-z));
        return s * fmaf(z, 1.0f - s, 1.0f);
    } else if constexpr (ACT == CUDA_MATMUL_EPILOGUE_GELU) {
        // P(z) + z p(z), p the normal density
        float gauss;
        const float cdf = normal_cdf<FAST>(z, gauss);
        return fmaf(z * (0.5f * kGeluC), gauss, cdf);
    } else if constexpr (ACT == CUDA_MATMUL_EPILOGUE_GELU_TANH) {
        // s + z s (1 - s) 2 u'
        const float z2 = z * z;
        const float u = kGeluC * fmaf(kGeluA * z2, z, z);
        const float s = divide<FAST>(1.0f, 1.0f + exp_of<FAST>(-2.0f * u));
        const float du = kGeluC * fmaf(3.0f * kGeluA, z2, 1.0f);
        return fmaf(2.0f * z * s * (1.0f - s), du, s);
    } else
        return 1.0f;
}

// Calls f(integral_constant<int, ACT>) for the run-time activation.
template <typename F>
__device__ __forceinline__ void with_activation(int act, F f)
{
    switch (act) {
    case CUDA_MATMUL_EPILOGUE_TANH: f(std::integral_constant<int, CUDA_MATMUL_EPILOGUE_TANH>()); break;
    case CUDA_MATMUL_EPILOGUE_RELU: f(std::integral_constant<int, CUDA_MATMUL_EPILOGUE_RELU>()); break;
    case CUDA_MATMUL_EPILOGUE_SIGMOID: f(std::integral_constant<int, CUDA_MATMUL_EPILOGUE_SIGMOID>()); break;
    case CUDA_MATMUL_EPILOGUE_GELU: f(std::integral_constant<int, CUDA_MATMUL_EPILOGUE_GELU>()); break;
    case CUDA_MATMUL_EPILOGUE_GELU_TANH: f(std::integral_constant<int, CUDA_MATMUL_EPILOGUE_GELU_TANH>()); break;
    case CUDA_MATMUL_EPILOGUE_SILU: f(std::integral_constant<int, CUDA_MATMUL_EPILOGUE_SILU>()); break;
    default: f(std::integral_constant<int, CUDA_MATMUL_EPILOGUE_NONE>()); break;
    }
}

} // namespace ptg
