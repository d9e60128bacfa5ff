// Activations of the gated feed-forward block and their derivatives, in fp32.
//     silu       g s(g)                 s the logistic function
//     gelu       g P(g)                 P the normal distribution function
//     gelu_tanh  g s(2 z), z = sqrt(2/pi) (g + 0.044715 g^3)   ( = g (1 + tanh z) / 2 )
// Each is written so that nothing cancels for large negative g, where act(g) goes to 0.
#pragma once

#include "fp4.cuh"

namespace i4l {

constexpr float kGeluC = 0.7978845608028654f;  // sqrt(2 / pi)
constexpr float kGeluA = 0.044715f;

// Two ulp of exp and of the reciprocal: the result is rounded to 16 bits.  (exp overflows to infinity for
// v < -88, whose reciprocal is the 0 that is wanted.)
__device__ __forceinline__ float logistic(float v) { return __fdividef(1.0f, 1.0f + __expf(-v)); }
// The normal distribution function and exp(-v^2 / 2), by the rational form 7.1.26 of Abramowitz and Stegun,
// "Handbook of Mathematical Functions": erfc(x) = (a1 t + ... + a5 t^5) exp(-x^2), t = 1 / (1 + p x), absolute error
// at most 1.5e-7, which is that of 1 + erf in fp32; the tail is not the difference of two near values.  (With erfcf
// the epilogue, not the products, set the time of a gated call: 302 against 183 us at 4096 x 14336 x 4096.)
__device__ __forceinline__ float normal_cdf(float v, float& density)
{
    density = __expf(-0.5f * v * v);
    const float t = __fdividef(1.0f, 1.0f + 0.3275911f * 0.7071067811865476f * fabsf(v));
    float q = fmaf(t, 1.061405429f, -1.453152027f);
    q = fmaf(t, q, 1.421413741f);
    q = fmaf(t, q, -0.284496736f);
    q = fmaf(t, q, 0.254829592f);
    q *= 0.5f * t * density;
    return v < 0.0f ? q : 1.0f - q;
}

template <int kAct>
__device__ __forceinline__ float gate_act(float g)
{
    if constexpr (kAct == kActSilu) return g * logistic(g);
    else if constexpr (kAct == kActGelu) { float density; return g * normal_cdf(g, density); }
    else return g * logistic(2.0f * kGeluC * (g + kGeluA * g * g * g));
}

// act(g) and act'(g).
template <int kAct>
__device__ __forceinline__ void gate_act_slope(float g, float& act, float& slope)
{
    if constexpr (kAct == kActSilu) {
        const float s = logistic(g);
        act = g * s;
        slope = s * (1.0f + g * logistic(-g));
    } else if constexpr (kAct == kActGelu) {
        float density;
        const float p = normal_cdf(g, density);
        act = g * p;
        slope = fmaf(g * 0.3989422804014327f, density, p);
    } else {
        const float z2 = 2.0f * kGeluC * (g + kGeluA * g * g * g);
        const float s = logistic(z2);
        act = g * s;
        slope = s * (1.0f + g * logistic(-z2) * 2.0f * kGeluC * (1.0f + 3.0f * kGeluA * g * g));
    }
}

}  // namespace i4l
