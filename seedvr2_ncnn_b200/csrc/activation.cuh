// Activations of the linear and group norm epilogues (S2_ACT_*), on fp32
// values held as pairs (packed f32x2 arithmetic).
//
// x sigmoid(t) = x / (1 + e^-t): no cancellation, so the error stays at a few
// units of 2^-24 of the result for any t, bf16 results included: what is rounded
// to bf16 is far smaller than x where x is negative, and an absolute error of x's
// size would show.  Further out e^-t becomes infinite and the result zero; at
// -inf it is the NaN of -inf times zero.
//
// Two special-function operations a value (an SM starts 16 a clock) and little
// else.  Four values that share one reciprocal need 1.25, and seven instructions
// more for products and for an exponent that stays in range: 8,000 x 2,560 x
// 1,024 with fp32 results and tanh GELU 76 us so and 88 shared, 6 x 14,400 x 512
// group norm with SiLU 55 and 55, but 60,000 x 1,024 x 256 in bf16 with SiLU 86
// and 80.
#pragma once

#include <cuda_runtime.h>

#include "../../include/seedvr2_cuda.h"

namespace s2 {

__device__ __forceinline__ float rcp_approx(float x)
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float ex2_approx(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float2 splat(float v)
{
    return make_float2(v, v);
}

constexpr double kSqrt2OverPi = 0.7978845608028654;
constexpr double kGeluCubic = 0.044715;
constexpr double kLog2e = 1.4426950408889634;

// 0.5 x (1 + erf(x / sqrt 2)) without a branch (erff's two branches cost a warp
// both, one element after another): with a = |x| and q = erfc(a / sqrt 2) / 2,
// the result is max(x, 0) - a q, so that negative x, where 1 + erf cancels, keep
// their digits.  q = r P(6 r - 1) e^(-a^2 / 2) with r = 1 / (a + 3): a + 3 takes
// out the scaled erfc's 1 / a, and the argument of P runs over (-0.63, 1].  P: the
// polynomial of degree 8 with the least relative error over 0 <= a <= 13.3 (4e-8;
// beyond, e^(-a^2 / 2) is zero), found by reweighted least squares.  Rounding
// leaves q within (20 + 2 x^2) 2^-24 of itself.  a above 30 is held there (no inf
// times zero); x / 2 + |x| / 2 keeps NaN and +inf.
__device__ __forceinline__ float2 gelu_erf(float2 x)
{
    constexpr float c[9] = {0.729083657f,  0.50933224f,     0.230019256f,   0.0472572222f,  -0.0104795201f,
                            -0.00692950143f, 0.0010774869f, 0.000911422248f, -0.000272206293f};
    const float2 ax = make_float2(fabsf(x.x), fabsf(x.y));
    const float2 neg = make_float2(fmaxf(-ax.x, -30.f), fmaxf(-ax.y, -30.f)); // -a
    const float2 d = __ffma2_rn(neg, splat(-1.f), splat(3.f));
    const float2 r = make_float2(rcp_approx(d.x), rcp_approx(d.y));
    const float2 s = __ffma2_rn(r, splat(6.f), splat(-1.f));
    float2 q = splat(c[8]);
#pragma unroll
    for (int i = 7; i >= 0; i--) q = __ffma2_rn(q, s, splat(c[i]));
    const float2 z2 = __fmul2_rn(__fmul2_rn(neg, splat((float)(-0.5 * kLog2e))), neg);
    q = __fmul2_rn(__fmul2_rn(q, r), make_float2(ex2_approx(z2.x), ex2_approx(z2.y)));
    const float2 positive = __ffma2_rn(x, splat(0.5f), __fmul2_rn(ax, splat(0.5f))); // max(x, 0), exact
    return __ffma2_rn(q, neg, positive);
}

// v = act(v)
template <int ACT, int N>
__device__ __forceinline__ void activate(float2 (&v)[N])
{
    if constexpr (ACT == S2_ACT_GELU_ERF)
    {
#pragma unroll
        for (int j = 0; j < N; j++) v[j] = gelu_erf(v[j]);
    }
    else if constexpr (ACT != S2_ACT_NONE)
    {
#pragma unroll
        for (int j = 0; j < N; j++)
        {
            const float2 x = v[j];
            float2 t; // -t log2(e)
            if constexpr (ACT == S2_ACT_SILU)
                t = __fmul2_rn(x, splat((float)-kLog2e));
            else
            {
                // 0.5 x (1 + tanh(w)) = x sigmoid(2w), w = sqrt(2/pi) (x + 0.044715 x^3)
                constexpr double k = -2 * kLog2e * kSqrt2OverPi; // each factor rounded once
                t = __fmul2_rn(x, __ffma2_rn(__fmul2_rn(x, splat((float)(k * kGeluCubic))), x, splat((float)k)));
            }
            const float2 d = __fadd2_rn(make_float2(ex2_approx(t.x), ex2_approx(t.y)), splat(1.f));
            v[j] = __fmul2_rn(x, make_float2(rcp_approx(d.x), rcp_approx(d.y)));
        }
    }
}

// The same of N values, the activation given at run time.
template <int N>
__device__ __forceinline__ void activate(float (&v)[N], int act)
{
    if (act == S2_ACT_NONE) return;
    constexpr int P = (N + 1) / 2;
    float2 p[P];
#pragma unroll
    for (int j = 0; j < P; j++) p[j] = make_float2(v[2 * j], 2 * j + 1 < N ? v[(2 * j + 1) % N] : 0.f);
    if (act == S2_ACT_SILU)
        activate<S2_ACT_SILU>(p);
    else if (act == S2_ACT_GELU_TANH)
        activate<S2_ACT_GELU_TANH>(p);
    else
        activate<S2_ACT_GELU_ERF>(p);
#pragma unroll
    for (int j = 0; j < N; j++) v[j] = j & 1 ? p[j / 2].y : p[j / 2].x;
}

} // namespace s2
