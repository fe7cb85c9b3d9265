// Element types of the entry points that take more than f32 (vxg_dtype), and exact / round-to-nearest-even
// conversions to and from f32 for vectors of eight elements.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "common.h"

namespace vxg {

template <int DT>
struct Elem;
template <>
struct Elem<VXG_DT_F16> {
  using type = __half;
  static __device__ __forceinline__ float widen(type v) { return __half2float(v); }
  static __device__ __forceinline__ type narrow(float v) { return __float2half_rn(v); }
};
template <>
struct Elem<VXG_DT_BF16> {
  using type = __nv_bfloat16;
  static __device__ __forceinline__ float widen(type v) { return __bfloat162float(v); }
  static __device__ __forceinline__ type narrow(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Elem<VXG_DT_F32> {
  using type = float;
  static __device__ __forceinline__ float widen(type v) { return v; }
  static __device__ __forceinline__ type narrow(float v) { return v; }
};

inline size_t dtype_bytes(int dt) { return dt == VXG_DT_F32 ? 4 : 2; }
inline bool dtype_known(int dt) { return dt == VXG_DT_F16 || dt == VXG_DT_BF16 || dt == VXG_DT_F32; }

// Two packed 16-bit elements <-> two floats.
template <int DT>
__device__ __forceinline__ float2 widen2(uint32_t w) {
  if constexpr (DT == VXG_DT_BF16) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  } else {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
}
template <int DT>
__device__ __forceinline__ uint32_t narrow2(float a, float b) {
  if constexpr (DT == VXG_DT_BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

// Eight consecutive elements, 16-byte aligned (16-bit types: one 16-byte access, f32: two).
template <int DT>
__device__ __forceinline__ void load8(const typename Elem<DT>::type* p, float (&v)[8]) {
  if constexpr (DT == VXG_DT_F32) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float2 f = widen2<DT>(w[i]);
      v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
  }
}
template <int DT>
__device__ __forceinline__ void store8(typename Elem<DT>::type* p, const float (&v)[8]) {
  if constexpr (DT == VXG_DT_F32) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(narrow2<DT>(v[0], v[1]), narrow2<DT>(v[2], v[3]),
                                              narrow2<DT>(v[4], v[5]), narrow2<DT>(v[6], v[7]));
  }
}

// Eight elements as they lie in memory.
template <int DT>
struct Raw {
  uint4 w[DT == VXG_DT_F32 ? 2 : 1];
};
template <int DT>
__device__ __forceinline__ void unpack(const Raw<DT>& r, float (&v)[8]) {
  if constexpr (DT == VXG_DT_F32) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      v[4 * i] = __uint_as_float(r.w[i].x), v[4 * i + 1] = __uint_as_float(r.w[i].y);
      v[4 * i + 2] = __uint_as_float(r.w[i].z), v[4 * i + 3] = __uint_as_float(r.w[i].w);
    }
  } else {
    const uint32_t w[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float2 f = widen2<DT>(w[i]);
      v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
  }
}

// f(std::integral_constant<int, DT>()) for a runtime element type that dtype_known() accepted.
template <class F>
inline void with_dtype(int dt, F&& f) {
  switch (dt) {
    case VXG_DT_F16: f(std::integral_constant<int, VXG_DT_F16>()); break;
    case VXG_DT_BF16: f(std::integral_constant<int, VXG_DT_BF16>()); break;
    default: f(std::integral_constant<int, VXG_DT_F32>()); break;
  }
}

}  // namespace vxg
