// Element types of the operators that take more than fp16, and vectors of them.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

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

// VEC elements that are loaded and stored at once (16 or 8 bytes, or one element).
template <class T, int VEC>
struct alignas(sizeof(T) * VEC) Vec {
  T v[VEC];
};
template <class T, int VEC>
__device__ __forceinline__ Vec<T, VEC> load_vec(const T* p) {
  Vec<T, VEC> r;
  if constexpr (sizeof(r) == 16) *reinterpret_cast<uint4*>(&r) = *reinterpret_cast<const uint4*>(p);
  else if constexpr (sizeof(r) == 8) *reinterpret_cast<uint2*>(&r) = *reinterpret_cast<const uint2*>(p);
  else r.v[0] = *p;
  return r;
}
template <class T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const Vec<T, VEC>& r) {
  if constexpr (sizeof(r) == 16) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&r);
  else if constexpr (sizeof(r) == 8) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(&r);
  else *p = r.v[0];
}

// fp32 arithmetic on the elements of a Vec: pairs in one instruction each (fma.rn.f32x2 and its kin), or one value where VEC
// is 1.  A pair costs one issue slot instead of two, and issue slots are what bounds the kernels that use these.
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 split(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 add(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 mul(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ float add(float a, float b) { return a + b; }
__device__ __forceinline__ float mul(float a, float b) { return a * b; }
__device__ __forceinline__ float fma(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ float total(float a) { return a; }
__device__ __forceinline__ float total(F2 a) {
  const float2 u = split(a);
  return u.x + u.y;
}
template <class F>
__device__ __forceinline__ F splat(float v) {
  if constexpr (sizeof(F) == 4) return v;
  else return f2(v, v);
}
template <int VEC>
struct Lanes {
  using F = F2;
  static constexpr int N = VEC / 2;
};
template <>
struct Lanes<1> {
  using F = float;
  static constexpr int N = 1;
};
// Two 16-bit values of one word, widened; and back.
template <class T>
__device__ __forceinline__ F2 widen2(uint32_t w) {
  if constexpr (std::is_same_v<T, __half>) {
    const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&w));
    return f2(u.x, u.y);
  } else {
    return f2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));   // bf16 is the upper half of an fp32
  }
}
template <class T>
__device__ __forceinline__ uint32_t narrow2(F2 a) {
  const float2 u = split(a);
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 h = __floats2half2_rn(u.x, u.y);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(u.x, u.y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <class T, int VEC>
__device__ __forceinline__ void widen(const Vec<T, VEC>& u, typename Lanes<VEC>::F (&out)[Lanes<VEC>::N]) {
  if constexpr (VEC == 1) {
    out[0] = to_f32(u.v[0]);
  } else if constexpr (sizeof(u) == 8) {
    const uint2 q = *reinterpret_cast<const uint2*>(&u);
    out[0] = widen2<T>(q.x), out[1] = widen2<T>(q.y);
  } else {
    const uint4 q = *reinterpret_cast<const uint4*>(&u);
    if constexpr (sizeof(T) == 4) {
      out[0] = f2(__uint_as_float(q.x), __uint_as_float(q.y)), out[1] = f2(__uint_as_float(q.z), __uint_as_float(q.w));
    } else {
      out[0] = widen2<T>(q.x), out[1] = widen2<T>(q.y), out[2] = widen2<T>(q.z), out[3] = widen2<T>(q.w);
    }
  }
}
template <class T, int VEC>
__device__ __forceinline__ Vec<T, VEC> narrow(const typename Lanes<VEC>::F (&in)[Lanes<VEC>::N]) {
  Vec<T, VEC> r;
  if constexpr (VEC == 1) {
    r.v[0] = from_f32<T>(in[0]);
  } else if constexpr (sizeof(r) == 8) {
    *reinterpret_cast<uint2*>(&r) = make_uint2(narrow2<T>(in[0]), narrow2<T>(in[1]));
  } else {
    uint4 q;
    if constexpr (sizeof(T) == 4) {
      const float2 a = split(in[0]), b = split(in[1]);
      q = make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
    } else {
      q = make_uint4(narrow2<T>(in[0]), narrow2<T>(in[1]), narrow2<T>(in[2]), narrow2<T>(in[3]));
    }
    *reinterpret_cast<uint4*>(&r) = q;
  }
  return r;
}

// A parameter vector (weight, bias) that is held in the activations' type or in fp32.
template <class T>
struct Param {
  const void* p;   // null: absent
  int f32;
  __device__ __forceinline__ float at(long long i) const {
    return f32 ? static_cast<const float*>(p)[i] : to_f32(static_cast<const T*>(p)[i]);
  }
  // VEC values from index i on; `absent` where there is no vector
  template <int VEC>
  __device__ __forceinline__ void get(long long i, float absent, typename Lanes<VEC>::F (&out)[Lanes<VEC>::N]) const {
    using F = typename Lanes<VEC>::F;
    if (!p) {
#pragma unroll
      for (int j = 0; j < Lanes<VEC>::N; ++j) out[j] = splat<F>(absent);
    } else if constexpr (VEC == 1) {
      out[0] = at(i);
    } else if (f32) {
#pragma unroll
      for (int j = 0; j < VEC; j += 4) {
        const float4 u = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i + j);
        out[j / 2] = f2(u.x, u.y), out[j / 2 + 1] = f2(u.z, u.w);
      }
    } else {
      widen<T, VEC>(load_vec<T, VEC>(static_cast<const T*>(p) + i), out);
    }
  }
};

__host__ inline int type_bytes(int dtype) { return dtype == BXL_F32 ? 4 : 2; }
__host__ inline bool known_type(int dtype) { return dtype == BXL_F16 || dtype == BXL_BF16 || dtype == BXL_F32; }

}  // namespace bxl
