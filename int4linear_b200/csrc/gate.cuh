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

// 1 / v for v >= 1, to one unit in the last place; 0 from 2^126 on.
__device__ __forceinline__ float reciprocal(float v)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// 1 / (1 + exp(-v)).  __expf errs by 2 + 1.173 |v| units in the last place, the quotient by two: 2^-16.4 at -80, a fortieth of
// half a step of fp16.  From v = -87.3 on (a divisor above 2^126) it is 0, so g s(g) is 0 where it is below 2^-119: nothing in
// fp16, while bfloat16 still has values down to 2^-133.  The form below goes on to them, but three more instructions per
// value cost the product's epilogue a seventh of its time (1024 x 14336 x 2048 mxfp4 silu: 28.7 -> 32.7 us).
__device__ __forceinline__ float logistic(float v) { return __fdividef(1.0f, 1.0f + __expf(-v)); }
// The same and c = 1 - s, from the exponential of -|v|: neither cancels, nothing overflows, and the smaller one goes to 0 as
// the exponential does (with fewer bits below 2^-126, at -104 for good).
__device__ __forceinline__ float logistic(float v, float& c)
{
    const float e = exp2f(-1.44269504f * fabsf(v));  // log2(e)
    const float r = reciprocal(1.0f + e), er = e * r;
    c = v < 0.0f ? r : er;
    return v < 0.0f ? er : r;
}
// The normal distribution function and exp(-v^2 / 2).  The lower tail is the density times t P(t), t = 1 / (1 + 0.362 |v|),
// P the polynomial of degree 6 for which the largest RELATIVE error against erfc(|v| / sqrt 2) / 2 is least over [0, 14.6]
// (weighted least squares, the weights multiplied by the error until it levels out: Lawson, "Contributions to the theory of
// linear least maximum approximation", 1961): 0.9e-6, 1.2e-6 evaluated in fp32, a four-hundredth of half a step of fp16.  So
// g P(g) keeps its bits as far out as the density does.  (With erfcf the epilogue, not the products, set the time of a
// gated call: 302 us at 4096 x 14336 x 4096.)
__device__ __forceinline__ float normal_cdf(float v, float& density)
{
    const float z = v * 0.84932180f;  // sqrt(log2(e) / 2)
    density = exp2f(-z * z);
    const float t = reciprocal(fmaf(0.362f, fabsf(v), 1.0f));
    float q = fmaf(t, 0.0476089977f, -0.178899616f);
    q = fmaf(t, q, 0.175130531f);
    q = fmaf(t, q, 0.029837992f);
    q = fmaf(t, q, 0.139068753f);
    q = fmaf(t, q, 0.142753929f);
    q = fmaf(t, q, 0.144499421f);
    q *= t * density;
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
        float c;
        const float s = logistic(g, c);
        act = g * s;
        slope = s * (1.0f + g * c);
    } else if constexpr (kAct == kActGelu) {
        float density;
        const float p = normal_cdf(g, density);
        act = g * p;
        slope = fmaf(g * 0.3989422804014327f, density, p);
    } else {
        const float z2 = 2.0f * kGeluC * (g + kGeluA * g * g * g);
        float c;
        const float s = logistic(z2, c);
        act = g * s;
        // Beyond +-32 the slope is 0 or 1 (so are s and c); the factor between them must not overflow there.
        const float near = fminf(fmaxf(g, -32.0f), 32.0f);
        slope = s * (1.0f + near * c * 2.0f * kGeluC * (1.0f + 3.0f * kGeluA * near * near));
    }
}

}  // namespace i4l
