// Activations of the gated feed-forward block and their derivatives, fp32.
//   silu:  act = g s,        act' = s (1 + g (1 - s)),                          s = 1 / (1 + e^-g)
//   gelu:  act = g s,        act' = s + 2 g s (1 - s) c (1 + 3 a g^2),          s = 1 / (1 + e^(-2 c (g + a g^3)))
//          (the tanh form: (1 + tanh z) / 2 = 1 / (1 + e^-2z)), c = sqrt(2 / pi), a = 0.044715
// Both are one exponential and one division. e^-z overflowing to infinity gives s = 0; neither form
// subtracts nearly equal numbers, so the relative error stays at a few fp32 steps and vanishes
// in the rounding to bf16.
#pragma once

#include "mt_common.cuh"

namespace mt {

static inline bool gated_act_known(int act) { return act == MT_ACT_SILU || act == MT_ACT_GELU; }

#if defined(__CUDACC__)

constexpr float GELU_C = 0.7978845608028654f;   // sqrt(2 / pi)
constexpr float GELU_A = 0.044715f;

__device__ __forceinline__ float gated_sigmoid(float z) { return __fdividef(1.0f, 1.0f + __expf(-z)); }

template <int kAct>
__device__ __forceinline__ float gated_act(float g) {
  if (kAct == MT_ACT_SILU) return g * gated_sigmoid(g);
  return g * gated_sigmoid(2.0f * GELU_C * g * fmaf(GELU_A * g, g, 1.0f));
}

// act(g) and act'(g)
template <int kAct>
__device__ __forceinline__ void gated_act_grad(float g, float& act, float& grad) {
  if (kAct == MT_ACT_SILU) {
    const float s = gated_sigmoid(g);
    act = g * s;
    grad = s * fmaf(g, 1.0f - s, 1.0f);
  } else {
    const float s = gated_sigmoid(2.0f * GELU_C * g * fmaf(GELU_A * g, g, 1.0f));
    act = g * s;
    grad = fmaf(act * (1.0f - s), 2.0f * GELU_C * fmaf(3.0f * GELU_A * g, g, 1.0f), s);
  }
}

#endif  // __CUDACC__

}  // namespace mt
