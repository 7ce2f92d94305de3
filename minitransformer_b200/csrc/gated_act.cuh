// Activations of the gated feed-forward block and their derivatives, fp32.
//   silu:  act = g s,        act' = s (1 + g (1 - s)),                          s = 1 / (1 + e^-g)
//   gelu:  act = g s,        act' = s + 2 g s (1 - s) c (1 + 3 a g^2),          s = 1 / (1 + e^(-2 c (g + a g^3)))
//          (the tanh form: (1 + tanh z) / 2 = 1 / (1 + e^-2z)), c = sqrt(2 / pi), a = 0.044715
// Both are one exponential and one division. e^-z overflowing to infinity gives s = 0; neither form
// subtracts nearly equal numbers, so the relative error stays at a few fp32 steps and vanishes
// in the rounding to bf16.
#pragma once

#include "quantize_common.cuh"

namespace mt {

static inline bool gated_act_known(int act) { return act == MT_ACT_SILU || act == MT_ACT_GELU; }

#if defined(__CUDACC__)

constexpr float GELU_C = 0.7978845608028654f;   // sqrt(2 / pi)
constexpr float GELU_A = 0.044715f;

__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float LOG2E = 1.4426950408889634f;
// 1 / (1 + e^-z), e^-z = 2^(-z log2 e)
__device__ __forceinline__ float gated_sigmoid(float z) { return rcp_approx(1.0f + ex2_approx(-LOG2E * z)); }

template <int kAct>
__device__ __forceinline__ float gated_act(float g) {
  if (kAct == MT_ACT_SILU) return g * gated_sigmoid(g);
  return g * gated_sigmoid(2.0f * GELU_C * g * fmaf(GELU_A * g, g, 1.0f));
}

// The gate limited to +-16, where gelu's s (1 - s) has long vanished in fp32 (z = 318); a NaN stays one.
__device__ __forceinline__ float gelu_limit(float g) {
  float y;
  asm("min.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(y) : "f"(g), "f"(16.0f));
  return y;
}

// act(g) and act'(g) of two values at once. gelu takes z and its slope, both cubic, of the limited gate: the slope of
// the gate itself leaves fp32 beyond |g| = 1e13, and infinity times an s (1 - s) of zero is a NaN where act' is 0 or 1.
template <int kAct>
__device__ __forceinline__ void gated_act_grad2(f32x2_t g, f32x2_t& act, f32x2_t& grad) {
  const f32x2_t one = pack2(1.0f, 1.0f);
  f32x2_t z, slope = g;
  if (kAct == MT_ACT_SILU) {
    z = mul2(g, pack2(-LOG2E, -LOG2E));
  } else {
    constexpr float C = 2.0f * GELU_C, CL = -LOG2E * 2.0f * GELU_C;
    float g0, g1;
    unpack2(g, g0, g1);
    const f32x2_t gl = pack2(gelu_limit(g0), gelu_limit(g1)), gg = mul2(gl, gl);
    z = mul2(gl, fma2(gg, pack2(CL * GELU_A, CL * GELU_A), pack2(CL, CL)));
    slope = mul2(gl, fma2(gg, pack2(3.0f * C * GELU_A, 3.0f * C * GELU_A), pack2(C, C)));
  }
  float z0, z1, s0, s1;
  unpack2(z, z0, z1);
  unpack2(add2(pack2(ex2_approx(z0), ex2_approx(z1)), one), s0, s1);
  const f32x2_t s = pack2(rcp_approx(s0), rcp_approx(s1));
  act = mul2(g, s);
  grad = mul2(s, fma2(slope, sub2(one, s), one));   // s + slope s (1 - s)
}

#endif  // __CUDACC__

}  // namespace mt
