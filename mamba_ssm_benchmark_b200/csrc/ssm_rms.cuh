// ssm_rms.cuh — what the forward and backward of the root-mean-square norm with a residual share.
//
//   t = x + residual,  n = t rstd,  y = n w,   rstd = (mean(t^2) + eps)^-1/2 over a row's C values
// t is a result, kept in the residual's type (the wider of the two), and what is normed: n comes from the rounded t, so
// that a backward that reads t sees the forward's values.
//
// Memory bounds both directions.  A team of 1 to 8 warps holds a row in registers, K vectors of VEC values a
// thread, and walks over rows; the rows ahead are on their way through slots of shared memory that only the thread
// that reads them writes (cp.async, no barrier, no registers).  Sums are fp32: at most 32 values in a thread, then a
// butterfly, then the warps in order.  Rows that no team holds take the kernels that pass over a row again.
#pragma once

#include <cuda_fp8.h>

#include <algorithm>
#include <initializer_list>

#include "ssm_b200.h"
#include "ssm_launch.cuh"
#include "ssm_vec.cuh"

namespace ssm {

constexpr int kRmsThreads = 256;    // of a CTA
constexpr int kRmsMost = 32;        // values of a row in a thread
constexpr int kRmsChain = 256;      // rows that one fp32 sum of the weight's gradient takes; what joins them is fp64
constexpr float kE4m3Max = 448.0f;
constexpr float kRmsTiny = 1e-30f;  // rows whose largest value is below it share its scale: 1 / scale stays finite

struct RmsParams {
  const void *x, *r, *w;              // r and w may be null
  void *y, *t;                        // t iff r
  long long xs, rs, ys, ts;           // row strides
  float* scale;                       // e4m3 only
  long long rows;
  int C, wbf16;
  float eps, inv_c;
  int norm;                           // 0: y = x, quantised
  // backward: t above is the normed sum, dy in y's place
  const void *dt;                     // gradient that arrives at t, or null
  void *dx, *dr;                      // dr null: the same tensor as dx
  long long dts, dxs, drs;
  float* part;                        // partial rows of the weight's gradient, or null
};

// B bytes into shared memory, zeros unless ok; asynchronously where the hardware can (not two bytes).
template <int B>
__device__ __forceinline__ void fetch_piece(void* dst, const void* src, bool ok) {
  if constexpr (B == 2)
    *static_cast<uint16_t*>(dst) = ok ? *static_cast<const uint16_t*>(src) : (uint16_t)0;
  else if constexpr (B == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(ok ? 16 : 0) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(smem_u32(dst)), "l"(src), "n"(B), "r"(ok ? B : 0)
                 : "memory");
}
// A thread's slot of VEC values of T: units of at most 16 bytes, the same unit of all threads side by side.
template <typename T, int VEC>
struct Slot {
  static constexpr int kBytes = VEC * (int)sizeof(T), kUnit = kBytes > 16 ? 16 : kBytes, kStep = kUnit / (int)sizeof(T);
  static __device__ __forceinline__ void fetch(unsigned char* at, const T* src, bool ok) {
#pragma unroll
    for (int i = 0; i < VEC / kStep; ++i) fetch_piece<kUnit>(at + (i * kRmsThreads + threadIdx.x) * kUnit, src + i * kStep, ok);
  }
  static __device__ __forceinline__ void read(const unsigned char* at, float (&v)[VEC]) {
#pragma unroll
    for (int i = 0; i < VEC / kStep; ++i) {
      float part[kStep];
      vec_load<T, kStep>(reinterpret_cast<const T*>(at + (i * kRmsThreads + threadIdx.x) * kUnit), part);
#pragma unroll
      for (int j = 0; j < kStep; ++j) v[i * kStep + j] = part[j];
    }
  }
};
__device__ __forceinline__ void queue_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void queue_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <typename T, int VEC>
__device__ __forceinline__ void write_piece(T* dst, const float (&v)[VEC]) {
  constexpr int kStep = VEC * sizeof(T) > 16 ? 16 / sizeof(T) : VEC;
#pragma unroll
  for (int i = 0; i < VEC; i += kStep) {
    float part[kStep];
#pragma unroll
    for (int j = 0; j < kStep; ++j) part[j] = v[i + j];
    vec_store<T, kStep>(dst + i, part);
  }
}
// VEC values to e4m3, nearest even; NaN stays NaN.
template <int VEC>
__device__ __forceinline__ void write_e4m3(uint8_t* dst, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    dst[0] = __nv_cvt_float_to_fp8(v[0], __NV_SATFINITE, __NV_E4M3);
  } else {
    uint16_t h[VEC / 2];
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i)
      h[i] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * i], v[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
    if constexpr (VEC == 8) {
      *reinterpret_cast<uint2*>(dst) = make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16);
    } else if constexpr (VEC == 4) {
      *reinterpret_cast<uint32_t*>(dst) = h[0] | (uint32_t)h[1] << 16;
    } else {
      *reinterpret_cast<uint16_t*>(dst) = h[0];
    }
  }
}

template <int VEC>
__device__ __forceinline__ void load_weight(const RmsParams& p, int c, float (&w)[VEC]) {
  if (p.w == nullptr) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) w[v] = 1.0f;
  } else if (p.wbf16) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) w[v] = to_f32(static_cast<const __nv_bfloat16*>(p.w)[c + v]);
  } else {
#pragma unroll
    for (int v = 0; v < VEC; ++v) w[v] = static_cast<const float*>(p.w)[c + v];
  }
}

// The warps that share a row: `wpr` of a CTA's.  Sums alternate between two buffers: a thread that reads one is at most
// one barrier behind those that write the other.
struct Team {
  int wpr, id, lane, warp, tid, size, turn;
  float2* red;                          // (2, wpr) of this team
  __device__ Team(int wpr_, float2* buf) : wpr(wpr_), turn(0) {
    lane = threadIdx.x & 31;
    const int w = threadIdx.x >> 5;
    id = w / wpr;
    warp = w - id * wpr;
    size = wpr * 32;
    tid = warp * 32 + lane;
    red = buf + id * 2 * wpr;
  }
  template <typename F>
  __device__ __forceinline__ float2 join(float2 v, F f) {
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1)
      v = f(v, make_float2(__shfl_xor_sync(0xffffffffu, v.x, m), __shfl_xor_sync(0xffffffffu, v.y, m)));
    if (wpr > 1) {
      float2* at = red + turn * wpr;
      turn ^= 1;
      if (lane == 0) at[warp] = v;
      asm volatile("bar.sync %0, %1;" ::"r"(1 + id), "r"(size) : "memory");
      v = at[0];
      for (int i = 1; i < wpr; ++i) v = f(v, at[i]);
    }
    return v;
  }
  __device__ __forceinline__ float2 sum(float a, float b) {
    return join(make_float2(a, b), [](float2 u, float2 v) { return make_float2(u.x + v.x, u.y + v.y); });
  }
  __device__ __forceinline__ float max(float a) {
    return join(make_float2(a, 0.0f), [](float2 u, float2 v) { return make_float2(fmaxf(u.x, v.x), 0.0f); }).x;
  }
};

// Stages of a thread's queue of `bytes` bytes a row.
constexpr int rms_depth(int bytes) { return bytes <= 48 ? 4 : bytes <= 256 ? 3 : 2; }

// ---- host -----------------------------------------------------------------------------------
inline long long rms_ceil(long long a, long long b) { return (a + b - 1) / b; }

// Warps to a row and vectors a thread, or k = 0: no team holds the row.  The fewest warps whose threads take at most
// `most` vectors: more rows side by side, fewer barriers.
struct RmsForm {
  int wpr, k;
};
inline RmsForm rms_form(long long C, int vec, int most) {
  for (int wpr = 1; wpr <= kRmsThreads / 32; wpr *= 2) {
    const long long k = rms_ceil(rms_ceil(C, vec), 32 * wpr);
    if (k <= most) return {wpr, (int)k};
  }
  return {0, 0};
}

// A tensor whose rows a kernel reads or writes in vectors.
struct RmsSide {
  const void* ptr;
  long long stride;
  int bytes;
};
int rms_vec(long long C, int xbytes, std::initializer_list<RmsSide> sides);
int rms_check(int64_t rows, int64_t C, const ssm_view& x, const ssm_view& residual, const void* weight, int32_t wdtype);

}  // namespace ssm
