// Activations of the linear layers and their derivatives, in fp32 on the unrounded pre-activation, one value or a pair (F2) at
// a time.
//
// silu, quick_gelu and gelu with tanh are z sigmoid(u), since (1 + tanh(u / 2)) / 2 = sigmoid(u); they take the fast
// exponential (2^-22 of its value) and reciprocal (2^-23).  With the roundings of 1 + exp(-u) and of the pair's products (4 2^-24) that is at
// most 2^-20 of the value, and |u| 2^-22 more on the left, where the value follows exp(u): the argument is rounded up to four times.
// At the clamp, |u| = 41.6, it comes to 2^-16.6; half a step of an fp16 result is 2^-11.  Beyond, the bound is absolute, as is that of
// gelu with erf, which takes the normal distribution's tail below: |z| 1e-7.  Factors that stand beside a vanishing one are clamped, so that infinite
// pre-activations give the limits (0 and z; derivatives 0 and 1; to 2^-50, as sigmoids end at 2^-60) and not 0 * inf.  A NaN
// reaches the result through other factors: what goes into a reciprocal, which a pair shares, never holds one (min_num), as it would
// make the neighbouring column NaN too.
#pragma once
#include "bxl_types.cuh"

namespace bxl {

__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// ... and the number, where `a` is NaN
__device__ __forceinline__ float min_num(float a, float b) { return fminf(a, b); }
__device__ __forceinline__ float magnitude(float a) { return fabsf(a); }
__device__ __forceinline__ float if_negative(float z, float a, float b) { return z < 0.f ? a : b; }
// ... and of pairs, for what has no instruction for two
#define BXL_ON_PAIRS(name)                                             \
  __device__ __forceinline__ F2 name(F2 a) {                           \
    const float2 u = split(a);                                         \
    return f2(name(u.x), name(u.y));                                   \
  }
BXL_ON_PAIRS(exp2_approx)
BXL_ON_PAIRS(magnitude)
#undef BXL_ON_PAIRS
// Both reciprocals of a pair from that of the product, which must be finite: one special-function instruction instead of two.
__device__ __forceinline__ F2 rcp_approx(F2 a) {
  const float2 u = split(a);
  const float r = rcp_approx(u.x * u.y);
  return mul(f2(u.y, u.x), f2(r, r));
}
__device__ __forceinline__ F2 min_nan(F2 a, float b) {
  const float2 u = split(a);
  return f2(min_nan(u.x, b), min_nan(u.y, b));
}
__device__ __forceinline__ F2 min_num(F2 a, float b) {
  const float2 u = split(a);
  return f2(min_num(u.x, b), min_num(u.y, b));
}
__device__ __forceinline__ F2 max_nan(F2 a, float b) {
  const float2 u = split(a);
  return f2(max_nan(u.x, b), max_nan(u.y, b));
}
__device__ __forceinline__ F2 if_negative(F2 z, F2 a, F2 b) {
  const float2 u = split(z), v = split(a), w = split(b);
  return f2(if_negative(u.x, v.x, w.x), if_negative(u.y, v.y, w.y));
}

// Phi(-|z|) of the normal distribution, `a` = |z| up to a bound beyond which it vanishes, by Abramowitz and Stegun, Handbook of
// Mathematical Functions, 7.1.26: with t = 1 / (1 + p y), erfc(y) = t (a1 + t (a2 + t (a3 + t (a4 + t a5)))) exp(-y^2) + error,
// |error| <= 1.5e-7, at y = a / sqrt(2).
// One reciprocal and one exponential, which the density takes too (`e` = exp(-z^2 / 2)).
template <class F>
__device__ __forceinline__ F normal_tail(F z, F a, F& e) {
  const F t = rcp_approx(fma(splat<F>(0.3275911f * 0.70710678118654752f), a, splat<F>(1.f)));
  e = exp2_approx(mul(mul(z, z), splat<F>(-0.72134752044448170f)));   // log2(e) / 2
  F p = fma(t, splat<F>(0.5f * 1.061405429f), splat<F>(0.5f * -1.453152027f));
  p = fma(t, p, splat<F>(0.5f * 1.421413741f));
  p = fma(t, p, splat<F>(0.5f * -0.284496736f));
  p = fma(t, p, splat<F>(0.5f * 0.254829592f));
  return mul(mul(p, t), e);
}
// exp(-u) of sigmoid(u) = 1 / (1 + exp(-u)), at most 2^60 (and that of a NaN), so that the product of two divisors is finite
template <int ACT, class F>
__device__ __forceinline__ F exp_minus_argument(F z) {
  constexpr float kLog2e = 1.4426950408889634f;
  F u;
  if constexpr (ACT == BXL_ACT_SILU) u = mul(z, splat<F>(-kLog2e));
  else if constexpr (ACT == BXL_ACT_QUICK_GELU) u = mul(z, splat<F>(-1.702f * kLog2e));
  else  // gelu with tanh: u = 2 sqrt(2 / pi) (z + 0.044715 z^3)
    u = mul(z, fma(mul(z, z), splat<F>(-0.07135481627260025f * kLog2e), splat<F>(-1.5957691216057308f * kLog2e)));
  return exp2_approx(min_num(u, 60.f));
}

template <int ACT, class F>
__device__ __forceinline__ F act_value(F z) {
  if constexpr (ACT == BXL_ACT_NONE) {
    return z;
  } else if constexpr (ACT == BXL_ACT_RELU) {
    return max_nan(z, 0.f);
  } else if constexpr (ACT == BXL_ACT_GELU) {
    // z Phi(z) = max(z, 0) - |z| Phi(-|z|): nothing cancels on either side
    const F a = min_num(magnitude(z), 1e3f);
    F e;
    const F q = normal_tail(z, a, e);
    return fma(mul(a, splat<F>(-1.f)), q, max_nan(z, 0.f));
  } else {
    return mul(max_nan(z, -1e3f), rcp_approx(add(exp_minus_argument<ACT>(z), splat<F>(1.f))));
  }
}

template <int ACT, class F>
__device__ __forceinline__ F act_slope(F z) {
  if constexpr (ACT == BXL_ACT_NONE) {
    return splat<F>(1.f);
  } else if constexpr (ACT == BXL_ACT_RELU) {
    // 0 or 1; 0 * z keeps a NaN
    const F zero = mul(min_nan(max_nan(z, -1.f), 1.f), splat<F>(0.f));
    return add(zero, if_negative(mul(z, splat<F>(-1.f)), splat<F>(1.f), splat<F>(0.f)));
  } else if constexpr (ACT == BXL_ACT_GELU) {
    // Phi(z) + z phi(z): of s = Phi(-a) - a phi(a) it is s on the left and 1 - s on the right
    const F a = min_num(magnitude(z), 1e3f);
    F e;
    const F q = normal_tail(z, a, e);
    const F s = fma(mul(a, splat<F>(-0.3989422804014327f)), e, q);
    return if_negative(z, s, fma(s, splat<F>(-1.f), splat<F>(1.f)));
  } else {
    // s + z s (1 - s) du/dz with 1 - s = s exp(-u), which is exact on both sides; beyond the clamps s (1 - s) vanishes
    constexpr float kEnd = ACT == BXL_ACT_GELU_TANH ? 12.f : 64.f;
    const F zc = min_nan(max_nan(z, -kEnd), kEnd), e = exp_minus_argument<ACT>(z);
    const F s = rcp_approx(add(e, splat<F>(1.f)));
    const F rest = mul(mul(zc, s), mul(s, e));
    if constexpr (ACT == BXL_ACT_SILU) return add(s, rest);
    else if constexpr (ACT == BXL_ACT_QUICK_GELU) return fma(rest, splat<F>(1.702f), s);
    else return fma(rest, fma(mul(zc, zc), splat<F>(0.2140644488178008f), splat<F>(1.5957691216057308f)), s);
  }
}

// Calls f with the activation as a compile-time constant.
template <int ACT>
struct ActTag {
  static constexpr int value = ACT;
};
template <class Fn>
__host__ __device__ __forceinline__ void with_act(int act, Fn&& f) {
  switch (act) {
    case BXL_ACT_RELU: f(ActTag<BXL_ACT_RELU>{}); break;
    case BXL_ACT_SILU: f(ActTag<BXL_ACT_SILU>{}); break;
    case BXL_ACT_GELU: f(ActTag<BXL_ACT_GELU>{}); break;
    case BXL_ACT_GELU_TANH: f(ActTag<BXL_ACT_GELU_TANH>{}); break;
    case BXL_ACT_QUICK_GELU: f(ActTag<BXL_ACT_QUICK_GELU>{}); break;
    default: f(ActTag<BXL_ACT_NONE>{});
  }
}

}  // namespace bxl
