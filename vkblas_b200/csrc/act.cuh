// act.cuh -- activations of the gated block, in fp32.
//
// All are g times a weight s in [0, 1]: silu s = sigmoid(g), gelu s = Phi(g), the
// normal distribution function, and the tanh form s = sigmoid(2y) with
// y = sqrt(2/pi) (g + 0.044715 g^3), since (1 + tanh y) / 2 = sigmoid(2y).  They run in the
// epilogue of a product, between its tiles, so they are straight code on the fast
// exponential and reciprocal (no slow path to branch to): with expf, a division and
// normcdff a tile's epilogue took 6.6 us of the 6 us that K = 1024 leaves it.
// Relative errors stay below 2e-6 for |g| < 6 and 1e-5 beyond (the exponent's own
// rounding), against 2.4e-4 for half a step of fp16.
//
// Phi by a formula of this file's own: for x = |g| / sqrt 2 and t = 1 / (1 + 0.3 x),
// erfc(x) = e^(-x^2) t Q(t), Q the least-maximum fit of degree 8 to e^(x^2) erfc(x) / t
// on 0 <= x <= 10 (4.5e-8 relative), and Phi(-|g|) = erfc(x) / 2: no cancellation in the
// negative tail, where (1 + erf) / 2 has it.
#pragma once
#include "vkblas_b200.h"

namespace vkb {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float GELU_A = 0.7978845608028654f;      // sqrt(2 / pi)
constexpr float GELU_B = 0.044715f;

// 2^v and 1 / v by the hardware's approximations (2 and 1 units in the last place; denormal
// results are 0).
__device__ __forceinline__ float fast_exp2(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float fast_rcp(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

__device__ __forceinline__ float sigmoid(float v) { return fast_rcp(1.f + fast_exp2(-LOG2E * v)); }

// Phi(g), and e^(-g^2 / 2) on the way.
__device__ __forceinline__ float normal_cdf(float g, float& e) {
    const float t = fast_rcp(fmaf(fabsf(g), 0.3f * 0.70710678118654752f, 1.f));
    float q = -0.12952275574207306f;
    q = fmaf(q, t, 0.4855624735355377f);
    q = fmaf(q, t, -0.5122765898704529f);
    q = fmaf(q, t, 0.5477182865142822f);
    q = fmaf(q, t, -0.0946495532989502f);
    q = fmaf(q, t, 0.21492557227611542f);
    q = fmaf(q, t, 0.14833930134773254f);
    q = fmaf(q, t, 0.17071521282196045f);
    q = fmaf(q, t, 0.1691880077123642f);
    e = fast_exp2(g * g * (-0.5f * LOG2E));
    const float h = 0.5f * t * q * e;
    return g > 0.f ? 1.f - h : h;
}

template <int ACT>
__device__ __forceinline__ float act_fwd(float g) {
    float e;
    if constexpr (ACT == VKBLAS_ACT_SILU) return g * sigmoid(g);
    else if constexpr (ACT == VKBLAS_ACT_GELU) return g * normal_cdf(g, e);
    else return g * sigmoid(2.f * GELU_A * (g + GELU_B * g * g * g));
}

// a = act(g), d = act'(g)
template <int ACT>
__device__ __forceinline__ void act_both(float g, float& a, float& d) {
    if constexpr (ACT == VKBLAS_ACT_SILU) {
        const float s = sigmoid(g);
        a = g * s;
        d = s + a * (1.f - s);
    } else if constexpr (ACT == VKBLAS_ACT_GELU) {
        float e;
        const float c = normal_cdf(g, e);
        a = g * c;
        d = fmaf(g, e * 0.3989422804014327f, c);                   // 1 / sqrt(2 pi)
    } else {
        const float s = sigmoid(2.f * GELU_A * (g + GELU_B * g * g * g));
        a = g * s;
        // From |g| = 16 on s is 0 or 1 and d the same; g^2 would pass the range further out.
        d = fabsf(g) < 16.f ? s + a * (1.f - s) * 2.f * GELU_A * (1.f + 3.f * GELU_B * g * g) : s;
    }
}

}  // namespace vkb
