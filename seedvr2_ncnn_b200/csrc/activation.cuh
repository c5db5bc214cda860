// Activations of the linear and group norm epilogues (S2_ACT_*), on fp32
// values.  The sigmoid forms are written as a quotient with one exponential:
// x / (1 + e^-t) has no cancellation, so its error stays at a few units of
// 2^-24 of the result where an fp32 output keeps it; tanh.approx (error
// 2^-11) would show there.  x -> -inf gives 0 (the quotient's denominator
// overflows to inf before x does) and NaN stays NaN.
#pragma once

#include <cuda_runtime.h>

#include "../../include/seedvr2_cuda.h"

namespace s2 {

// x * sigmoid(t)
__device__ __forceinline__ float times_sigmoid(float x, float t)
{
    return __fdividef(x, 1.f + __expf(-t));
}

template <int ACT>
__device__ __forceinline__ float activate_one(float x)
{
    if (ACT == S2_ACT_SILU) return times_sigmoid(x, x);
    if (ACT == S2_ACT_GELU_TANH)
    {
        // 0.5 x (1 + tanh(u)) = x sigmoid(2u), u = sqrt(2/pi) (x + 0.044715 x^3)
        const float k = 2.f * 0.7978845608028654f;
        return times_sigmoid(x, k * x * (1.f + 0.044715f * x * x));
    }
    if (ACT == S2_ACT_GELU_ERF) return 0.5f * x * (1.f + erff(x * 0.70710678118654752f));
    return x;
}

// The activation is uniform over a launch: one branch per N values.
template <int N>
__device__ __forceinline__ void activate(float (&v)[N], int act)
{
    switch (act)
    {
    case S2_ACT_SILU:
#pragma unroll
        for (int j = 0; j < N; j++) v[j] = activate_one<S2_ACT_SILU>(v[j]);
        break;
    case S2_ACT_GELU_TANH:
#pragma unroll
        for (int j = 0; j < N; j++) v[j] = activate_one<S2_ACT_GELU_TANH>(v[j]);
        break;
    case S2_ACT_GELU_ERF:
#pragma unroll
        for (int j = 0; j < N; j++) v[j] = activate_one<S2_ACT_GELU_ERF>(v[j]);
        break;
    default: break;
    }
}

} // namespace s2
