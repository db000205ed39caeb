// The activations of a gated dense layer and their derivatives, for the kernels that apply them.
#pragma once
#include <math.h>

namespace tf {

// values of the `activation` argument (those of the activation operator, and two more)
enum { kGateSigmoid = 0, kGateRelu = 1, kGateTanh = 2, kGateSilu = 4, kGateGelu = 5 };
inline bool is_gate(int a) { return a >= 0 && a <= 5 && a != 3; }
// f(std::integral_constant) with the activation as a constant
template <class F> inline void with_gate(int a, F&& f) {
  switch (a) {
    case kGateSigmoid: f(std::integral_constant<int, kGateSigmoid>()); break;
    case kGateRelu: f(std::integral_constant<int, kGateRelu>()); break;
    case kGateTanh: f(std::integral_constant<int, kGateTanh>()); break;
    case kGateSilu: f(std::integral_constant<int, kGateSilu>()); break;
    default: f(std::integral_constant<int, kGateGelu>()); break;
  }
}

#ifdef __CUDACC__
// 1 / d of a d from 1 to 2: the fast quotient, within 2 units of the last place, and a step of Newton's method, which squares that error and leaves
// about one rounding.  (With the general division 6728 x 64 x 2720 forward with silu takes 112 us, 92 so.)
__device__ __forceinline__ float inverse(float d) {
  const float r = __fdividef(1.f, d);
  return fmaf(r, fmaf(-d, r, 1.f), r);
}
// 1 / (1 + exp(-g)) and one minus that, both without cancellation: exp of a number that is never positive
// FAST: the short road to the reciprocal.  Where a thread has one or two outputs the general one is as fast (64 x 784 x 256 forward 8.9 us, 8.4 so).
template <bool FAST = true> __device__ __forceinline__ void sigmoids(float g, float& s, float& rest) {
  const float e = expf(-fabsf(g)), r = FAST ? inverse(1.f + e) : 1.f / (1.f + e);
  s = g >= 0.f ? r : e * r;
  rest = g >= 0.f ? e * r : r;
}
template <int ACT, bool FAST = true> __device__ __forceinline__ float gate_value(float g) {
  if (ACT == kGateRelu) return g > 0.f || g != g ? g : 0.f;
  if (ACT == kGateTanh) return tanhf(g);
  if (ACT == kGateGelu) return g * (0.5f * erfcf(-0.70710678118654752f * g));
  float s, rest;
  sigmoids<FAST>(g, s, rest);
  return ACT == kGateSigmoid ? s : g * s;
}
__device__ __forceinline__ float gate_value_of(int activation, float g) {
  switch (activation) {
    case kGateSigmoid: return gate_value<kGateSigmoid>(g);
    case kGateRelu: return gate_value<kGateRelu>(g);
    case kGateTanh: return gate_value<kGateTanh>(g);
    case kGateSilu: return gate_value<kGateSilu>(g);
    default: return gate_value<kGateGelu>(g);
  }
}
// The activation's value and its derivative
template <int ACT> __device__ __forceinline__ void gate_slope(float g, float& value, float& slope) {
  if (ACT == kGateRelu) { value = gate_value<ACT>(g); slope = g > 0.f ? 1.f : g != g ? g : 0.f; return; }
  if (ACT == kGateTanh) {
    const float e = expf(-2.f * fabsf(g)), r = inverse(1.f + e);
    value = tanhf(g);
    slope = 4.f * e * r * r;                   // 1 - tanh^2 without the subtraction
    return;
  }
  if (ACT == kGateGelu) {
    const float below = 0.5f * erfcf(-0.70710678118654752f * g);
    value = g * below;
    slope = fmaf(g, 0.39894228040143268f * expf(-0.5f * g * g), below);
    return;
  }
  float s, rest;
  sigmoids(g, s, rest);
  value = ACT == kGateSigmoid ? s : g * s;
  slope = ACT == kGateSigmoid ? s * rest : fmaf(g * s, rest, s);
}
#endif

}  // namespace tf
