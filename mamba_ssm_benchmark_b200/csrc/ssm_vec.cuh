// ssm_vec.cuh — vectors of VEC consecutive elements (16 bytes, or one element) as float.
#pragma once

#include "ssm_common.cuh"

namespace ssm {

template <typename T, int VEC>
__device__ __forceinline__ void vec_load(const T* src, float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    v[0] = to_f32(src[0]);
  } else if constexpr (sizeof(T) == 4) {
    static_assert(VEC == 4, "fp32 vectors are 4 wide");
    load4(src, v);
  } else {
    static_assert(VEC == 8, "bf16 vectors are 8 wide");
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
    *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    uint4 q;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&q);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4*>(dst) = q;
  }
}

}  // namespace ssm
