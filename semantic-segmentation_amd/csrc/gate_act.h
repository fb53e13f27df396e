// Activations of the gated feed-forward unit and their derivatives (gated.hip, mx4.hip).
#pragma once
#include "common.h"

namespace ssmi {

enum { kSwish = 0, kGelu = 1, kRelu = 2, kSigmoid = 3 };

// exp of the bfloat16 variants: v_exp_f32 on x log2(e), relative error under 2^-20 for |x| < 16 - far below the output's 2^-9; the
// float32 variants take the library's
template <typename T>
__device__ __forceinline__ float gate_exp(float v) {
  if constexpr (sizeof(T) == 2) return __builtin_amdgcn_exp2f(v * 1.44269504f);
  return expf(v);
}
template <typename T>
__device__ __forceinline__ float gate_sigmoid(float v) {
  return __builtin_amdgcn_rcpf(1.f + gate_exp<T>(-v));      // exp = inf gives 0
}
// Phi(g) = (1 + erf(g / sqrt 2)) / 2, and exp(-g^2 / 2) beside it.  bfloat16: Abramowitz and Stegun 7.1.26, whose own exponential is the
// density's - erf off by at most 1.5e-7, one reciprocal, one exponential, seven multiply-adds (the library's erff costs far more instructions
// and the registers of both its branches); float32: the library's.
template <typename T>
__device__ __forceinline__ float gate_phi(float g, float& density) {
  density = gate_exp<T>(-0.5f * g * g);
  if constexpr (sizeof(T) == 2) {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f * 0.70710678f, fabsf(g), 1.f));
    float p = fmaf(1.061405429f, t, -1.453152027f);
    p = fmaf(p, t, 1.421413741f);
    p = fmaf(p, t, -0.284496736f);
    p = fmaf(p, t, 0.254829592f);
    const float upper = 0.5f * p * t * density;      // 1 - Phi(|g|)
    return g < 0.f ? upper : 1.f - upper;
  }
  return 0.5f * (1.f + erff(g * 0.70710678f));
}
template <typename T, int ACT>
__device__ __forceinline__ float gate_act(float g) {
  [[maybe_unused]] float density;
  if constexpr (ACT == kSwish) return g * gate_sigmoid<T>(g);
  if constexpr (ACT == kGelu) return g * gate_phi<T>(g, density);
  if constexpr (ACT == kRelu) return g < 0.f ? 0.f : g;      // a NaN stays one
  return gate_sigmoid<T>(g);
}
template <typename T, int ACT>
__device__ __forceinline__ void gate_act_both(float g, float& a, float& d) {
  if constexpr (ACT == kSwish) {
    const float s = gate_sigmoid<T>(g);
    a = g * s;
    d = s * (1.f + g * (1.f - s));
  } else if constexpr (ACT == kGelu) {
    float density;
    const float c = gate_phi<T>(g, density);
    a = g * c;
    d = c + g * 0.39894228f * density;
  } else if constexpr (ACT == kRelu) {
    a = g < 0.f ? 0.f : g;
    d = g > 0.f ? 1.f : 0.f;
  } else {
    a = gate_sigmoid<T>(g);
    d = a * (1.f - a);
  }
}

// runs body(integral constant) for the activation: one branch around an epilogue, none inside it
template <int V> struct ActIs { static constexpr int value = V; };
template <typename Body>
__device__ __forceinline__ void with_act(int act, Body body) {
  if (act == kSwish) body(ActIs<kSwish>{});
  else if (act == kGelu) body(ActIs<kGelu>{});
  else if (act == kRelu) body(ActIs<kRelu>{});
  else body(ActIs<kSigmoid>{});
}

}  // namespace ssmi
