// Activations of the linear layers and their derivatives, in fp32 on the unrounded pre-activation.
//
// The sigmoid forms (silu, quick_gelu, and gelu with tanh: z (1 + tanh(u/2)) / 2 = z sigmoid(u)) take the fast exponential
// and division, whose errors are 2^-21 of the value: far below the 2^-12 of an fp16 result.  Factors that stand beside a
// vanishing one are clamped first, so that infinite pre-activations give the limits (0, z; derivatives 0 and 1) and not
// 0 * inf; NaN stays NaN through the other factor.
#pragma once
#include "../../include/basedxl_b200.h"

namespace bxl {

__device__ __forceinline__ float sigmoid_f32(float u) { return __fdividef(1.f, 1.f + __expf(-u)); }
// u of gelu with tanh: 2 sqrt(2 / pi) (z + 0.044715 z^3)
__device__ __forceinline__ float gelu_tanh_argument(float z) { return z * fmaf(0.07135481627260025f * z, z, 1.5957691216057308f); }

template <int ACT>
__device__ __forceinline__ float act_value(float z) {
  const float zc = fmaxf(z, -1e30f);   // -inf * 0
  if constexpr (ACT == BXL_ACT_RELU) return z < 0.f ? 0.f : z;
  else if constexpr (ACT == BXL_ACT_SILU) return __fdividef(zc, 1.f + __expf(-z));
  else if constexpr (ACT == BXL_ACT_GELU) return 0.5f * zc * (1.f + erff(z * 0.70710678118654752f));
  else if constexpr (ACT == BXL_ACT_GELU_TANH) return __fdividef(zc, 1.f + __expf(-gelu_tanh_argument(z)));
  else if constexpr (ACT == BXL_ACT_QUICK_GELU) return __fdividef(zc, 1.f + __expf(-1.702f * z));
  else return z;
}

template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  const float zc = fminf(fmaxf(z, -1e3f), 1e3f);   // beyond it the factors beside it are exactly 0
  if constexpr (ACT == BXL_ACT_RELU) {
    return z > 0.f ? 1.f : z == z ? 0.f : z;
  } else if constexpr (ACT == BXL_ACT_GELU) {
    // Phi(z) + z phi(z)
    return fmaf(zc, 0.3989422804014327f * __expf(-0.5f * zc * zc), 0.5f * (1.f + erff(z * 0.70710678118654752f)));
  } else if constexpr (ACT == BXL_ACT_SILU) {
    const float s = sigmoid_f32(z);
    return fmaf(zc * s, 1.f - s, s);
  } else if constexpr (ACT == BXL_ACT_QUICK_GELU) {
    const float s = sigmoid_f32(1.702f * z);
    return fmaf(1.702f * zc * s, 1.f - s, s);
  } else if constexpr (ACT == BXL_ACT_GELU_TANH) {
    const float s = sigmoid_f32(gelu_tanh_argument(z));
    return fmaf(zc * s * (1.f - s), fmaf(0.2140644488178008f * zc, zc, 1.5957691216057308f), s);
  } else {
    return 1.f;
  }
}

// Calls f with the activation as a compile-time constant.
template <int ACT>
struct ActTag {
  static constexpr int value = ACT;
};
template <class F>
__host__ __device__ __forceinline__ void with_act(int act, F&& f) {
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
