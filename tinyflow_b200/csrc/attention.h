// Attention: arguments that its kernels share, what a query sees, and scores behind the product.
//
//   s_ij = scale q_i k_j,  c_ij = cap tanh(s_ij / cap) or s_ij,  z_ij = (c_ij - slope_h |i - j|) log2(e)
//   p_ij = 2^(z_ij - max) / sum over the keys j that query i sees,  o_i = sum_j p_ij v_j
//
// Query i of T_q stands at position i + T_k - T_q of the keys.  A query that sees no key has o = 0 and no gradient.
#pragma once
#include "common.h"

namespace tf {

struct AttentionArgs {
  const float *q, *k, *v;
  const float *documents, *prefix, *slopes;            // may be null
  const float *out, *dout;                             // backward
  float* stats;                                        // (max, 1 / sum) of every sequence, head and query, or null
  float *o, *dq, *dk, *dv;
  int B, H, G, group;                                  // sequences, query heads, key-value heads, query heads of one of those
  int Tq, Tk, D;
  int causal, window;                                  // window 0: none
  float scale, cap;                                    // cap 0: none
};

#ifdef __CUDACC__
constexpr float kLog2e = 1.4426950408889634f;

// Both of 2 ulp; below 2^-126 zero
__device__ __forceinline__ float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float reciprocal(float x) { float y; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

// Two numbers an instruction, rounded as each alone would be
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ unsigned long long pair_of(float2 v) { unsigned long long p; asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(v.x), "f"(v.y)); return p; }
__device__ __forceinline__ float2 of_pair(unsigned long long p) { float2 v; asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(p)); return v; }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(pair_of(a)), "l"(pair_of(b)), "l"(pair_of(c)));
  return of_pair(d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(pair_of(a)), "l"(pair_of(b)));
  return of_pair(d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(pair_of(a)), "l"(pair_of(b)));
  return of_pair(d);
}
__device__ __forceinline__ float2 at2(const float* v, int k) { return make_float2(v[k], v[k + 1]); }
__device__ __forceinline__ void put2(float* v, int k, float2 x) { v[k] = x.x; v[k + 1] = x.y; }

// The keys of a query at position `at`: those of [lo, hi] and those before `prefix`, if of its document.
struct Sight { int lo, hi; };
__device__ __forceinline__ Sight sight_of(const AttentionArgs& a, int at) {
  Sight s;
  s.hi = a.causal ? at : a.window ? (int)min((long long)at + a.window - 1, (long long)a.Tk - 1) : a.Tk - 1;
  s.lo = a.window ? max(at - a.window + 1, 0) : 0;
  return s;
}
__device__ __forceinline__ int prefix_of(const AttentionArgs& a, int b) {
  if (!a.prefix) return 0;
  const float p = __ldg(a.prefix + b);
  return p > 0.f ? (p < (float)a.Tk ? (int)ceilf(p) : a.Tk) : 0;
}
// The document of the token at position `at`; -1: of none
__device__ __forceinline__ float document_of(const AttentionArgs& a, int b, int at) {
  return at >= 0 && at < a.Tk ? __ldg(a.documents + (int64_t)b * a.Tk + at) : -1.f;
}
__device__ __forceinline__ bool sees(const Sight& s, int prefix, int j) { return (j >= s.lo && j <= s.hi) || j < prefix; }
__device__ __forceinline__ float max_of_finite_or(float m) { return m == -INFINITY ? 0.f : m; }        // of a row that has seen nothing
#endif

}  // namespace tf
