// ssm_rms.cuh — what the forward and backward of the root-mean-square norm with a residual share.
//
//   t = x + residual,  n = t rstd,  y = n w,   rstd = (mean(t^2) + eps)^-1/2 over a row's C values
// t is a result, kept in the residual's type (the wider of the two), and what is normed: n comes from the rounded t, so
// that a backward that reads t sees the forward's values.
//
// Memory bounds both directions.  A team of 1 to 16 warps holds a row in registers, K vectors of VEC values a
// thread, and walks over rows; the rows ahead are on their way through slots of shared memory that only the thread
// that reads them writes (cp.async, no barrier, no registers).  Sums are fp32: at most 16 values in a thread, then a
// butterfly over the warp and one over the warps.  Rows that no team holds take the kernels that pass over a row again; a thread
// has more than 16 values there and joins sums of four in fp64 (in one fp32 chain a row of 2^24 equal values was off by 2^-13).
#pragma once

#include <cuda_fp8.h>

#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "ssm_b200.h"
#include "ssm_launch.cuh"
#include "ssm_rows.cuh"

namespace ssm {

constexpr int kRmsMost = 16;        // values of a row in a thread: with more, registers leave too few rows to an SM
constexpr int kRmsWarps = 16;       // of a team, at most
constexpr int kRmsThreads = 32 * kRmsWarps;
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
  int wide8;                          // e4m3 rows start at multiples of 8
  // backward: t above is the normed sum, dy in y's place
  const void *dt;                     // gradient that arrives at t, or null
  void *dx, *dr;                      // dr null: the same tensor as dx
  long long dts, dxs, drs;
  float* part;                        // partial rows of the weight's gradient, or null
};

// A CTA's queue to zeros, for what fetch does not write.
__device__ __forceinline__ void clear_queue(unsigned char* queue, int bytes) {
  for (int i = threadIdx.x * 16; i < bytes; i += blockDim.x * 16) *reinterpret_cast<uint4*>(queue + i) = make_uint4(0, 0, 0, 0);
  __syncthreads();
}
__device__ __forceinline__ void queue_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void queue_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// VEC values to e4m3, nearest even (NaN stays NaN), the first n of them to dst; wide: dst is aligned to VEC bytes.
template <int VEC>
__device__ __forceinline__ void write_e4m3(uint8_t* dst, int n, bool wide, const float2 (&v)[VEC / 2]) {
  uint16_t h[VEC / 2];
#pragma unroll
  for (int i = 0; i < VEC / 2; ++i) h[i] = __nv_cvt_float2_to_fp8x2(v[i], __NV_SATFINITE, __NV_E4M3);
  if (wide && n >= VEC) {
    if constexpr (VEC == 8)
      *reinterpret_cast<uint2*>(dst) = make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16);
    else
      *reinterpret_cast<uint32_t*>(dst) = h[0] | (uint32_t)h[1] << 16;
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i < n) dst[i] = (uint8_t)(h[i / 2] >> (i & 1 ? 8 : 0));
  }
}

// The weight to L2 while the kernel before still runs; the grid's first threads take a line each.
__device__ __forceinline__ void prefetch_weight(const RmsParams& p) {
  const long long at = ((long long)blockIdx.x * blockDim.x + threadIdx.x) * 128;
  if (p.w != nullptr && at < (long long)p.C * (p.wbf16 ? 2 : 4)) prefetch_l2(static_cast<const char*>(p.w) + at);
}
// The first n of VEC weights from channel c on; zeros behind.
template <int VEC>
__device__ __forceinline__ void load_weight(const RmsParams& p, int c, int n, float2 (&w)[VEC / 2]) {
  auto one = [&](int v) {
    if (v >= n) return 0.0f;
    return p.w == nullptr ? 1.0f
           : p.wbf16      ? to_f32(static_cast<const __nv_bfloat16*>(p.w)[c + v])
                          : static_cast<const float*>(p.w)[c + v];
  };
#pragma unroll
  for (int v = 0; v < VEC / 2; ++v) w[v] = make_float2(one(2 * v), one(2 * v + 1));
}
__device__ __forceinline__ float weight_at(const RmsParams& p, int c) {
  if (p.w == nullptr) return 1.0f;
  return p.wbf16 ? to_f32(static_cast<const __nv_bfloat16*>(p.w)[c]) : static_cast<const float*>(p.w)[c];
}

// f(c, n) for the channels c, c + 512 .. of this one of a CTA's threads: n (a constant) of them at once, four and the rest singly.
template <typename F>
__device__ __forceinline__ void by_fours(int C, F f) {
  int c = threadIdx.x;
  for (; c + 3 * kRmsThreads < C; c += 4 * kRmsThreads) f(c, std::integral_constant<int, 4>());
  for (; c < C; c += kRmsThreads) f(c, std::integral_constant<int, 1>());
}

// The warps that share a row: `wpr` of a CTA's.  Results of the warps alternate between two buffers: a thread that reads
// one is at most one barrier behind those that write the other.
struct Team {
  int wpr, id, lane, warp, tid, size, turn;
  float2* red;                          // (2, kRmsWarps) of this team
  __device__ Team(int wpr_, float2* buf) : wpr(wpr_), turn(0) {
    lane = threadIdx.x & 31;
    const int w = threadIdx.x >> 5;
    id = w / wpr;
    warp = w - id * wpr;
    size = wpr * 32;
    tid = warp * 32 + lane;
    red = buf + id * 2 * kRmsWarps;
  }
  // every warp's value, in lane i that of warp i (`none` past the last)
  __device__ __forceinline__ float2 exchange(float2 v, float2 none) {
    float2* at = red + turn;
    turn ^= kRmsWarps;
    if (lane == 0) at[warp] = v;
    asm volatile("bar.sync %0, %1;" ::"r"(1 + id), "r"(size) : "memory");
    return lane < wpr ? at[lane] : none;
  }
  template <int LANES>
  static __device__ __forceinline__ float2 add(float2 v) {
#pragma unroll
    for (int m = LANES / 2; m >= 1; m /= 2)
      v = add2(v, make_float2(__shfl_xor_sync(0xffffffffu, v.x, m), __shfl_xor_sync(0xffffffffu, v.y, m)));
    return v;
  }
  __device__ __forceinline__ float2 sum(float2 v) {
    v = add<32>(v);
    if (wpr == 1) return v;
    v = add<16>(exchange(v, make_float2(0.0f, 0.0f)));        // lanes 0 .. 15 hold the warps'
    return make_float2(__shfl_sync(0xffffffffu, v.x, 0), __shfl_sync(0xffffffffu, v.y, 0));
  }
  __device__ __forceinline__ float sum(float v) {
#pragma unroll
    for (int m = 16; m >= 1; m /= 2) v += __shfl_xor_sync(0xffffffffu, v, m);
    if (wpr == 1) return v;
    v = exchange(make_float2(v, 0.0f), make_float2(0.0f, 0.0f)).x;
#pragma unroll
    for (int m = 8; m >= 1; m /= 2) v += __shfl_xor_sync(0xffffffffu, v, m);
    return __shfl_sync(0xffffffffu, v, 0);
  }
  // of numbers that are not negative, which compare as their bits do
  __device__ __forceinline__ float max(float v) {
    uint32_t b = __reduce_max_sync(0xffffffffu, __float_as_uint(v));
    if (wpr > 1) {
      const float2 zero = make_float2(0.0f, 0.0f);
      b = __reduce_max_sync(0xffffffffu, __float_as_uint(exchange(make_float2(__uint_as_float(b), 0.0f), zero).x));
    }
    return __uint_as_float(b);
  }
};
constexpr int kRmsRed = 2 * kRmsWarps * 8;       // floats2 of at most eight teams

// Rows on their way to a team: with more, fewer CTAs share an SM and wait for one another's barriers (16384 x 5120 bf16
// backward: 179 us with four rows, 141 with three, 137 with two).
constexpr int kRmsDepth = 2;

// ---- host -----------------------------------------------------------------------------------
inline long long rms_ceil(long long a, long long b) { return (a + b - 1) / b; }

// Warps to a row and vectors a thread (one of `ks`, the largest first), or k = 0: no team holds the row.  The form that
// wastes the fewest lanes (2560 bf16 values: five warps of two vectors), with the fewest warps.
struct RmsForm {
  int wpr, k;
  int teams() const { return std::max(1, 8 / wpr); }     // rows side by side in a CTA
  int threads() const { return 32 * wpr * teams(); }
};
inline RmsForm rms_form(long long C, int vec, std::initializer_list<int> ks) {
  RmsForm f = {0, 0};
  for (int k : ks) {
    const long long wpr = rms_ceil(C, 32LL * vec * k);
    if (wpr <= kRmsWarps && (f.k == 0 || wpr * k < (long long)f.wpr * f.k)) f = {(int)wpr, k};
  }
  return f;
}

// A tensor whose rows a kernel reads or writes in units of 16 bytes.
struct RmsSide {
  const void* ptr;
  long long stride;
  int bytes;
};
bool rms_aligned(long long C, int vec, std::initializer_list<RmsSide> sides);
int rms_check(int64_t rows, int64_t C, const ssm_view& x, const ssm_view& residual, const void* weight, int32_t wdtype);

}  // namespace ssm
