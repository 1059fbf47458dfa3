// act.cuh -- activations of the gated block, in fp32.
//
// All are g times a weight s in [0, 1]: silu s = sigmoid(g), gelu s = Phi(g)
// (normcdff keeps its relative accuracy in the negative tail, where
// (1 + erf) / 2 cancels), and the tanh form s = sigmoid(2y) with
// y = sqrt(2/pi) (g + 0.044715 g^3), since (1 + tanh y) / 2 = sigmoid(2y).
#pragma once
#include "vkblas_b200.h"

namespace vkb {

constexpr float GELU_A = 0.7978845608028654f;      // sqrt(2 / pi)
constexpr float GELU_B = 0.044715f;

__device__ __forceinline__ float sigmoid(float v) { return 1.f / (1.f + expf(-v)); }

template <int ACT>
__device__ __forceinline__ float act_fwd(float g) {
    if constexpr (ACT == VKBLAS_ACT_SILU) return g * sigmoid(g);
    else if constexpr (ACT == VKBLAS_ACT_GELU) return g * normcdff(g);
    else return g * sigmoid(2.f * GELU_A * (g + GELU_B * g * g * g));
}

// a = act(g), d = act'(g)
template <int ACT>
__device__ __forceinline__ void act_both(float g, float& a, float& d) {
    if constexpr (ACT == VKBLAS_ACT_SILU) {
        const float s = sigmoid(g);
        a = g * s;
        d = s + g * s * (1.f - s);
    } else if constexpr (ACT == VKBLAS_ACT_GELU) {
        const float c = normcdff(g);
        a = g * c;
        d = c + g * expf(-0.5f * g * g) * 0.3989422804014327f;     // 1 / sqrt(2 pi)
    } else {
        const float s = sigmoid(2.f * GELU_A * (g + GELU_B * g * g * g));
        a = g * s;
        d = s + g * s * (1.f - s) * 2.f * GELU_A * (1.f + 3.f * GELU_B * g * g);
    }
}

}  // namespace vkb
