// ssm_vec.cuh — vectors of VEC consecutive elements (up to 16 bytes, aligned to their size) as float.
#pragma once

#include "ssm_common.cuh"

namespace ssm {

template <typename T, int VEC>
__device__ __forceinline__ void vec_load(const T* src, float (&v)[VEC]) {
  constexpr int kBytes = VEC * (int)sizeof(T);
  static_assert(kBytes <= 16 && (VEC & (VEC - 1)) == 0, "a vector is one load");
  if constexpr (VEC == 1) {
    v[0] = to_f32(src[0]);
  } else if constexpr (sizeof(T) == 4) {
    if constexpr (VEC == 4) load4(src, v);
    else load2(src, v);
  } else if constexpr (VEC <= 4) {
    if constexpr (VEC == 4) load4(src, v);
    else load2(src, v);
  } else {
    const uint4 q = *reinterpret_cast<const uint4*>(src);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}

template <typename T, int VEC>
__device__ __forceinline__ void vec_store(T* dst, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    dst[0] = from_f32<T>(v[0]);
  } else if constexpr (sizeof(T) == 4) {
    if constexpr (VEC == 4) *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
    else *reinterpret_cast<float2*>(dst) = make_float2(v[0], v[1]);
  } else {
    uint32_t w[VEC / 2];
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    if constexpr (VEC == 8) *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (VEC == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(dst) = w[0];
  }
}

// VEC elements as they lie in memory: loaded now, widened later (a prefetch in half the registers).
template <typename T, int VEC>
struct alignas(VEC * sizeof(T)) Raw {
  T x[VEC];
  __device__ __forceinline__ void load(const T* src) { *this = *reinterpret_cast<const Raw*>(src); }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < VEC; ++i) x[i] = from_f32<T>(0.0f);
  }
  __device__ __forceinline__ void widen(float (&v)[VEC]) const {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = to_f32(x[i]);
  }
};

}  // namespace ssm
