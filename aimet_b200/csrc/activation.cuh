// The activations a linear layer can carry in its epilogue, and their slopes, in float32.
//
//   relu       max(z, 0)
//   gelu       z / 2 * (1 + erf(z / sqrt 2))
//   gelu_tanh  z / 2 * (1 + tanh(sqrt(2 / pi) * (z + 0.044715 z^3)))
//   silu       z / (1 + exp(-z))
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
        return 0.5f * z * (1.f + tanhf(0.79788456f * (z + 0.044715f * z * z * z)));
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
        if (fabsf(z) > 14.f)
            return z > 0.f ? 1.f : 0.f;
        return 0.5f * (1.f + erff(z * 0.70710678f)) + z * expf(-0.5f * z * z) * 0.39894228f;
    }
    else if constexpr (ACT == AQ_ACT_GELU_TANH)
    {
        if (fabsf(z) > 14.f)
            return z > 0.f ? 1.f : 0.f;
        const float t = tanhf(0.79788456f * (z + 0.044715f * z * z * z));
        return 0.5f * (1.f + t) + 0.5f * z * (1.f - t * t) * 0.79788456f * (1.f + 0.134145f * z * z);
    }
    else if constexpr (ACT == AQ_ACT_SILU)
    {
        if (fabsf(z) > 100.f)
            return z > 0.f ? 1.f : 0.f;
        const float p = 1.f / (1.f + expf(-z));
        return p * (1.f + z * (1.f - p));
    }
    else
        return 1.f;
}

// dz = dy * act'(z).  A zero slope gives zero whatever dy holds (a masked infinity stays out of the sums).
template <int ACT>
__device__ __forceinline__ float act_grad(float dy, float z)
{
    if constexpr (ACT == AQ_ACT_NONE)
        return dy;
    const float s = act_slope<ACT>(z);
    return s == 0.f ? 0.f : dy * s;
}

// f.template operator()<ACT>() for the run-time value `act`; every kernel launcher below dispatches through it
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
