// Activations of the gated feed-forward block and their derivatives, fp32.
//   silu:  act = g s,        act' = s (1 + g (1 - s)),                          s = 1 / (1 + e^-g)
//   gelu:  act = g s,        act' = s + 2 g s (1 - s) c (1 + 3 a g^2),          s = 1 / (1 + e^(-2 c (g + a g^3)))
//          (the tanh form: (1 + tanh z) / 2 = 1 / (1 + e^-2z)), c = sqrt(2 / pi), a = 0.044715
// Both are one exponential and one reciprocal, both approximate. The rounding of z shows in e^-z in proportion to |z|: s, and
// with it act, is off by at most (1 + |z|) 2^-20 of its value, and where s is subnormal by a step of 2^-149 on top. act' is
// the sum of two terms that cancel at its root (g near -1.28 with silu, -0.75 with gelu), and holds 1 - s, a multiple of
// 2^-24 for s near 1: its error is that share of the terms' magnitudes, not of their sum.
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
// s = 1 / (1 + e^-z) as far as fp32 reaches (2^-149), z below -88 included, where 1 + e^-z is not an fp32 number any more
// and s not a normal one: e^-z = t^2 with t = 2^(-z log2(e) / 2), and everything is scaled by 2^-32,
//   s = 2^-32 / (2^-32 + (2^-16 t)^2).
// (The scale in the exponent's argument instead would round away bits of it.)
constexpr float SIG_ARG = -0.5f * LOG2E, SIG_T = 0x1p-16f, SIG_S = 0x1p-32f;
__device__ __forceinline__ float gated_sigmoid(float z) {
  const float t = SIG_T * ex2_approx(SIG_ARG * z);
  return SIG_S * rcp_approx(fmaf(t, t, SIG_S));
}

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
    z = mul2(g, pack2(SIG_ARG, SIG_ARG));
  } else {
    constexpr float C = 2.0f * GELU_C, CL = SIG_ARG * 2.0f * GELU_C;
    float g0, g1;
    unpack2(g, g0, g1);
    const f32x2_t gl = pack2(gelu_limit(g0), gelu_limit(g1)), gg = mul2(gl, gl);
    z = mul2(gl, fma2(gg, pack2(CL * GELU_A, CL * GELU_A), pack2(CL, CL)));
    slope = mul2(gl, fma2(gg, pack2(3.0f * C * GELU_A, 3.0f * C * GELU_A), pack2(C, C)));
  }
  float z0, z1, s0, s1;
  unpack2(z, z0, z1);
  const f32x2_t t = mul2(pack2(ex2_approx(z0), ex2_approx(z1)), pack2(SIG_T, SIG_T)), unit = pack2(SIG_S, SIG_S);
  unpack2(fma2(t, t, unit), s0, s1);
  const f32x2_t s = mul2(pack2(rcp_approx(s0), rcp_approx(s1)), unit);
  act = mul2(g, s);
  grad = mul2(s, fma2(slope, sub2(one, s), one));   // s + slope s (1 - s)
}

#endif  // __CUDACC__

}  // namespace mt
