// Element types of the operators that take more than fp16, and vectors of them.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "../../include/basedxl_b200.h"

namespace bxl {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// VEC elements that are loaded and stored at once (16 bytes, or one element).
template <class T, int VEC>
struct alignas(sizeof(T) * VEC) Vec {
  T v[VEC];
};
template <class T, int VEC>
__device__ __forceinline__ Vec<T, VEC> load_vec(const T* p) {
  Vec<T, VEC> r;
  if constexpr (sizeof(r) == 16) *reinterpret_cast<uint4*>(&r) = *reinterpret_cast<const uint4*>(p);
  else r.v[0] = *p;
  return r;
}
template <class T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const Vec<T, VEC>& r) {
  if constexpr (sizeof(r) == 16) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&r);
  else *p = r.v[0];
}

// A parameter vector (weight, bias) that is held in the activations' type or in fp32.
template <class T>
struct Param {
  const void* p;   // null: absent
  int f32;
  __device__ __forceinline__ float at(long long i) const {
    return f32 ? static_cast<const float*>(p)[i] : to_f32(static_cast<const T*>(p)[i]);
  }
  template <int VEC>
  __device__ __forceinline__ void get(long long i, float (&out)[VEC]) const {
    if constexpr (VEC == 1) {
      out[0] = at(i);
    } else if (f32) {
#pragma unroll
      for (int j = 0; j < VEC; j += 4) {
        const float4 u = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i + j);
        out[j] = u.x, out[j + 1] = u.y, out[j + 2] = u.z, out[j + 3] = u.w;
      }
    } else {
      const Vec<T, VEC> u = load_vec<T, VEC>(static_cast<const T*>(p) + i);
#pragma unroll
      for (int j = 0; j < VEC; ++j) out[j] = to_f32(u.v[j]);
    }
  }
};

__host__ inline int type_bytes(int dtype) { return dtype == BXL_F32 ? 4 : 2; }
__host__ inline bool known_type(int dtype) { return dtype == BXL_F16 || dtype == BXL_BF16 || dtype == BXL_F32; }

}  // namespace bxl
