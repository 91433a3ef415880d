// The activations a linear layer can carry in its epilogue, and their slopes, in float32.
//
//   relu       max(z, 0)
//   gelu       z P(z),       P(z) = (1 + erf(z / sqrt 2)) / 2
//   gelu_tanh  z s(2 u(z)),  u(z) = sqrt(2 / pi) (z + 0.044715 z^3), s the logistic function: (1 + tanh u) / 2 = s(2 u)
//   silu       z s(z)
//
// The *2 functions are for 16-bit results: two float32 lanes at a time, the hardware's exponential and reciprocal (relative
// error near 2^-21), and for P the rational approximation 7.1.26 of Abramowitz and Stegun (Handbook of Mathematical
// Functions; error of erf at most 1.5e-7), whose exp(-z^2 / 2) is also the density that the slope needs.  With erff and
// expf the backward pass of a gelu layer is bound by instructions instead of memory: see grad_z_kernel.
//
// NaN stays NaN in every value.  The slopes take their limits 0 and 1 beyond |z| = 14 (gelu; what is left of the
// derivative is below 1e-40) or |z| = 100 (silu; below 1e-41): the formulas would form 0 * inf there.
#pragma once

#include "common.cuh"

namespace aq
{
template <int ACT>
__device__ __forceinline__ float act_value(float z)
{
    if constexpr (ACT == AQ_ACT_RELU)
        return z < 0.f ? 0.f : z;
    else if constexpr (ACT == AQ_ACT_GELU)
        return 0.5f * z * (1.f + erff(z * 0.70710678f));
    else if constexpr (ACT == AQ_ACT_GELU_TANH)
        return z / (1.f + expf(-1.5957691f * z * fmaf(0.044715f * z, z, 1.f)));
    else if constexpr (ACT == AQ_ACT_SILU)
        return z / (1.f + expf(-z));
    else
        return z;
}

template <int ACT>
__device__ __forceinline__ float act_slope(float z)
{
    if constexpr (ACT == AQ_ACT_RELU)
        return z > 0.f ? 1.f : 0.f;
    else if constexpr (ACT == AQ_ACT_GELU)
    {
        const float s = fmaf(z * 0.39894228f, expf(-0.5f * z * z), 0.5f * (1.f + erff(z * 0.70710678f)));
        return fabsf(z) > 14.f ? (z > 0.f ? 1.f : 0.f) : s;
    }
    else if constexpr (ACT == AQ_ACT_GELU_TANH)
    {
        const float z2 = z * z;
        const float p  = 1.f / (1.f + expf(-1.5957691f * z * fmaf(0.044715f, z2, 1.f)));
        const float s  = fmaf(z * p * (1.f - p), 1.5957691f * fmaf(0.134145f, z2, 1.f), p);
        return fabsf(z) > 14.f ? (z > 0.f ? 1.f : 0.f) : s;
    }
    else if constexpr (ACT == AQ_ACT_SILU)
    {
        const float p = 1.f / (1.f + expf(-z));
        const float s = p * fmaf(z, 1.f - p, 1.f);
        return fabsf(z) > 100.f ? (z > 0.f ? 1.f : 0.f) : s;
    }
    else
        return 1.f;
}

// dz = dy * act'(z).  Where relu is off the result is zero whatever dy holds (an infinity stays out of the sums).
template <int ACT>
__device__ __forceinline__ float act_grad(float dy, float z)
{
    if constexpr (ACT == AQ_ACT_NONE)
        return dy;
    if constexpr (ACT == AQ_ACT_RELU)
        return z > 0.f ? dy : 0.f;
    return dy * act_slope<ACT>(z);
}

// ---- two lanes, for 16-bit results --------------------------------------------------------------------------------
__device__ __forceinline__ f32x2_t splat2(float v)
{
    return pair(v, v);
}
__device__ __forceinline__ f32x2_t rcp2(f32x2_t v)
{
    float lo, hi;
    unpair(v, lo, hi);
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(lo));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(hi));
    return pair(lo, hi);
}
__device__ __forceinline__ f32x2_t exp2_2(f32x2_t v)
{
    float lo, hi;
    unpair(v, lo, hi);
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(lo));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(hi));
    return pair(lo, hi);
}
// |z| at most `most`; NaN stays
__device__ __forceinline__ f32x2_t clamp2(f32x2_t v, float most)
{
    float lo, hi;
    unpair(v, lo, hi);
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(lo) : "f"(most));
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(hi) : "f"(most));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(lo) : "f"(-most));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(hi) : "f"(-most));
    return pair(lo, hi);
}
__device__ __forceinline__ f32x2_t abs2(f32x2_t v)
{
    return v & 0x7fffffff7fffffffull;
}
// s(x) with x log2(e) given
__device__ __forceinline__ f32x2_t logistic2(f32x2_t x)
{
    return rcp2(add2(splat2(1.f), exp2_2(x ^ 0x8000000080000000ull)));
}
// P(z) and e = exp(-z^2 / 2): 7.1.26 at |z| / sqrt 2, so p / sqrt 2 = 0.23164189 and the five coefficients halved
__device__ __forceinline__ f32x2_t normal_cdf2(f32x2_t z, f32x2_t& e)
{
    const f32x2_t t = rcp2(fma2(splat2(0.23164189f), abs2(z), splat2(1.f)));
    f32x2_t q       = fma2(splat2(0.5307027145f), t, splat2(-0.7265760135f));
    q               = fma2(q, t, splat2(0.7107068705f));
    q               = fma2(q, t, splat2(-0.142248368f));
    q               = fma2(q, t, splat2(0.127414796f));
    e                  = exp2_2(mul2(mul2(z, splat2(-0.72134752f)), z));
    const f32x2_t tail = mul2(mul2(q, t), e), rest = sub2(splat2(1.f), tail);   // P(-|z|), P(|z|)
    // The tail itself for z < 0: taken from 1 it loses what it is small by (4 % off at z = -5, now 0.2 %).
    float z0, z1, t0, t1, r0, r1;
    unpair(z, z0, z1);
    unpair(tail, t0, t1);
    unpair(rest, r0, r1);
    return pair(z0 < 0.f ? t0 : r0, z1 < 0.f ? t1 : r1);
}

template <int ACT>
__device__ __forceinline__ f32x2_t act_value2(f32x2_t z)
{
    if constexpr (ACT == AQ_ACT_GELU)
    {
        f32x2_t e;
        return mul2(z, normal_cdf2(z, e));
    }
    else if constexpr (ACT == AQ_ACT_GELU_TANH)
        // 1.5957691 log2(e) = 2.3022082
        return mul2(z, logistic2(mul2(mul2(z, splat2(2.3022082f)), fma2(mul2(z, splat2(0.044715f)), z, splat2(1.f)))));
    else if constexpr (ACT == AQ_ACT_SILU)
        return mul2(z, logistic2(mul2(z, splat2(1.44269504f))));
    else
    {
        float lo, hi;
        unpair(z, lo, hi);
        return pair(act_value<ACT>(lo), act_value<ACT>(hi));
    }
}

// The activation of one value on its way to a result in T: the same function in every kernel.
template <typename T, int ACT>
__device__ __forceinline__ float act_as(float z)
{
    if constexpr (sizeof(T) == 4)
        return act_value<ACT>(z);
    float lo, hi;
    unpair(act_value2<ACT>(splat2(z)), lo, hi);
    return lo;
}

template <int ACT>
__device__ __forceinline__ f32x2_t act_grad2(f32x2_t dy, f32x2_t z)
{
    if constexpr (ACT == AQ_ACT_GELU)
    {
        f32x2_t e;
        z               = clamp2(z, 14.f);
        const f32x2_t p = normal_cdf2(z, e);
        return mul2(dy, fma2(mul2(z, splat2(0.39894228f)), e, p));
    }
    else if constexpr (ACT == AQ_ACT_GELU_TANH)
    {
        z                = clamp2(z, 14.f);
        const f32x2_t z2 = mul2(z, z);
        const f32x2_t p  = logistic2(mul2(mul2(z, splat2(2.3022082f)), fma2(z2, splat2(0.044715f), splat2(1.f))));
        const f32x2_t u  = fma2(z2, splat2(0.134145f * 1.5957691f), splat2(1.5957691f));
        return mul2(dy, fma2(mul2(mul2(z, p), sub2(splat2(1.f), p)), u, p));
    }
    else if constexpr (ACT == AQ_ACT_SILU)
    {
        z               = clamp2(z, 100.f);
        const f32x2_t p = logistic2(mul2(z, splat2(1.44269504f)));
        return mul2(dy, mul2(p, fma2(z, sub2(splat2(1.f), p), splat2(1.f))));
    }
    else
    {
        float d0, d1, z0, z1;
        unpair(dy, d0, d1);
        unpair(z, z0, z1);
        return pair(act_grad<ACT>(d0, z0), act_grad<ACT>(d1, z1));
    }
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
