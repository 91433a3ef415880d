// The activations a linear layer can carry in its epilogue, and their slopes, in float32.
//
//   relu       max(z, 0)
//   gelu       z P(z),       P(z) = (1 + erf(z / sqrt 2)) / 2
//   gelu_tanh  z s(2 u(z)),  u(z) = sqrt(2 / pi) (z + 0.044715 z^3), s the logistic function: (1 + tanh u) / 2 = s(2 u)
//   silu       z s(z)
//
// FAST is for 16-bit results: the hardware's exponential and reciprocal (relative error near 2^-21), and for P the
// rational approximation 7.1.26 of Abramowitz and Stegun (Handbook of Mathematical Functions; error of erf at most
// 1.5e-7), whose exp(-z^2 / 2) is also the density that the slope needs.  The backward pass of a 16384 x 11008 bf16
// layer is bound by instructions with erff and expf: see grad_z_kernel.
//
// NaN stays NaN in every value.  The slopes take their limits 0 and 1 beyond |z| = 14 (gelu; what is left of the
// derivative is below 1e-40) or |z| = 100 (silu; below 1e-41): the formulas would form 0 * inf there.
#pragma once

#include "common.cuh"

namespace aq
{
__device__ __forceinline__ float fast_rcp(float x)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float fast_exp2(float x)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// s(x) from -x log2(e)
template <bool FAST>
__device__ __forceinline__ float logistic(float x)
{
    if constexpr (FAST)
        return fast_rcp(1.f + fast_exp2(-1.44269504f * x));
    else
        return 1.f / (1.f + expf(-x));
}

// P(z), and exp(-z^2 / 2) for the slope
template <bool FAST>
__device__ __forceinline__ float normal_cdf(float z, float& e)
{
    if constexpr (FAST)
    {
        // 7.1.26 at |z| / sqrt 2: p / sqrt 2 = 0.23164189, the five coefficients halved
        const float t = fast_rcp(fmaf(0.23164189f, fabsf(z), 1.f));
        float q       = fmaf(0.5307027145f, t, -0.7265760135f);
        q             = fmaf(q, t, 0.7107068705f);
        q             = fmaf(q, t, -0.142248368f);
        q             = fmaf(q, t, 0.127414796f);
        e             = fast_exp2(-0.72134752f * z * z);
        const float tail = q * t * e;   // P(-|z|)
        return z > 0.f ? 1.f - tail : tail;
    }
    else
    {
        e = expf(-0.5f * z * z);
        return 0.5f * (1.f + erff(z * 0.70710678f));
    }
}

template <int ACT, bool FAST>
__device__ __forceinline__ float act_value(float z)
{
    if constexpr (ACT == AQ_ACT_RELU)
        return z < 0.f ? 0.f : z;
    else if constexpr (ACT == AQ_ACT_GELU)
    {
        float e;
        return z * normal_cdf<FAST>(z, e);
    }
    else if constexpr (ACT == AQ_ACT_GELU_TANH)
        return z * logistic<FAST>(1.5957691f * z * fmaf(0.044715f * z, z, 1.f));
    else if constexpr (ACT == AQ_ACT_SILU)
        return z * logistic<FAST>(z);
    else
        return z;
}

template <int ACT, bool FAST>
__device__ __forceinline__ float act_slope(float z)
{
    if constexpr (ACT == AQ_ACT_RELU)
        return z > 0.f ? 1.f : 0.f;
    else if constexpr (ACT == AQ_ACT_GELU)
    {
        float e;
        const float p = normal_cdf<FAST>(z, e);
        const float s = fmaf(z * 0.39894228f, e, p);
        return fabsf(z) > 14.f ? (z > 0.f ? 1.f : 0.f) : s;
    }
    else if constexpr (ACT == AQ_ACT_GELU_TANH)
    {
        const float z2 = z * z;
        const float p  = logistic<FAST>(1.5957691f * z * fmaf(0.044715f, z2, 1.f));
        const float s  = fmaf(z * p * (1.f - p), 1.5957691f * fmaf(0.134145f, z2, 1.f), p);
        return fabsf(z) > 14.f ? (z > 0.f ? 1.f : 0.f) : s;
    }
    else if constexpr (ACT == AQ_ACT_SILU)
    {
        const float p = logistic<FAST>(z);
        const float s = p * fmaf(z, 1.f - p, 1.f);
        return fabsf(z) > 100.f ? (z > 0.f ? 1.f : 0.f) : s;
    }
    else
        return 1.f;
}

// dz = dy * act'(z).  Where relu is off the result is zero whatever dy holds (an infinity stays out of the sums).
template <int ACT, bool FAST>
__device__ __forceinline__ float act_grad(float dy, float z)
{
    if constexpr (ACT == AQ_ACT_NONE)
        return dy;
    if constexpr (ACT == AQ_ACT_RELU)
        return z > 0.f ? dy : 0.f;
    return dy * act_slope<ACT, FAST>(z);
}

// f(std::integral_constant<int, ACT>) for the run-time value `act`
template <typename F>
inline int with_activation(int act, F&& f)
{
    switch (act)
    {
    case AQ_ACT_NONE: return f(std::integral_constant<int, AQ_ACT_NONE> {});
    case AQ_ACT_RELU: return f(std::integral_constant<int, AQ_ACT_RELU> {});
    case AQ_ACT_GELU: return f(std::integral_constant<int, AQ_ACT_GELU> {});
    case AQ_ACT_GELU_TANH: return f(std::integral_constant<int, AQ_ACT_GELU_TANH> {});
    case AQ_ACT_SILU: return f(std::integral_constant<int, AQ_ACT_SILU> {});
    default: return AQ_ERR_INVALID_ARG;
    }
}
}   // namespace aq
