// ssm_norm.cu — group norm over channels-last tensors with an activation and a gate, forward and
// backward.
//
//   n = (x - mean) rstd,  a = act(n w + b),  y = a silu(z)
// with mean (0 unless centred) and rstd = (var + eps)^-1/2 over the (positions, C / G) elements of
// every (sample, group).  One position per sample is the norm of every head of every token.
//
// Backward, with p = n w + b, e = dy silu(z) act'(p), M = positions C / G:
//   dz = dy a silu'(z);  dw = sum e n;  db = sum e
//   dx = rstd (e w - (s1 + n s2) / M),  s1 = sum_group e w (0 unless centred), s2 = sum_group e w n
//
// Memory bounds every form; which launch does what:
//   * one position ("rows"): one kernel, every tensor moved once.  1 to 32 lanes, or eight warps, share
//     a group, each lane holding K vectors of VEC channels in registers; sums are butterflies, mean and
//     variance two passes over registers.  Groups that do not fit (above 8192 channels) take the last form
//     with a warp per group for the sums.
//   * more positions: per-(slab of rows, channel) partial sums, a combine per (sample, group), an
//     element-wise pass (the tensors are read twice).
// Sums over at most kChain rows in a row are fp32, what joins them is fp64, all in a fixed order: no atomics, results are
// reproducible.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdio>
#include <initializer_list>

#include "ssm_b200.h"
#include "ssm_launch.cuh"
#include "ssm_vec.cuh"

namespace ssm {
int report_error(int code, const char* msg);
}  // namespace ssm

namespace {

using ssm::vec_load;
using ssm::vec_store;

constexpr int kWarps = 8;           // warps per CTA: rows taken side by side
// Rows that one fp32 sum takes: its roundings stay below kChain 2^-24 = 1.5e-5 of the sum of its terms' sizes however long
// the batch is (8192 rows in a row, as a batch of 65536 short samples had, came to 8e-5).
constexpr int kChain = 256;

struct NormParams {
  const void *x, *z, *dy;
  void *y, *dx, *dz;
  long long xs, xp, zs, zp, gs, gp;   // sample and position strides of x, z, dy
  long long ys, yp, dxs, dxp, dzs, dzp;
  const float *w, *b;
  float* stats;                       // (N, G, 2): mean, rstd
  float* sums;                        // (N, G, 2): s1, s2 of the backward
  float* part;                        // partial sums, see the kernels
  float *dw, *db;
  long long N, P, C;
  int G, cg;                          // groups, channels per group
  int nslab;                          // slabs of rows per sample (more positions) or of all rows
  long long slab;                     // rows per slab
  float eps;
  int center, silu, gate;
};

__device__ __forceinline__ float dsilu(float z, float s) { return s * fmaf(z, 1.0f - s, 1.0f); }

// y from the normalised values.  The activation and the gate are branched on once per vector, not per element
// (per element they made 39 instructions of 13).
template <int VEC>
__device__ __forceinline__ void norm_out(const NormParams& p, const float (&n)[VEC], const float (&w)[VEC],
                                         const float (&b)[VEC], const float (&z)[VEC], float (&y)[VEC]) {
#pragma unroll
  for (int v = 0; v < VEC; ++v) y[v] = fmaf(n[v], w[v], b[v]);
  if (p.silu) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) y[v] *= ssm::sigmoid(y[v]);
  }
  if (p.gate) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) y[v] *= z[v] * ssm::sigmoid(z[v]);
  }
}
// e = d loss / d (n w + b) in dy's place, and dz in z's.
template <int VEC>
__device__ __forceinline__ void norm_grad(const NormParams& p, const float (&n)[VEC], const float (&w)[VEC],
                                          const float (&b)[VEC], float (&z)[VEC], float (&dy)[VEC]) {
  float a[VEC], d[VEC];                  // act and act' of n w + b
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    a[v] = fmaf(n[v], w[v], b[v]);
    d[v] = 1.0f;
  }
  if (p.silu) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      const float s = ssm::sigmoid(a[v]);
      d[v] = dsilu(a[v], s);
      a[v] *= s;
    }
  }
  if (p.gate) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      const float s = ssm::sigmoid(z[v]), g = dy[v];
      dy[v] = g * (z[v] * s);
      z[v] = g * a[v] * dsilu(z[v], s);
    }
  }
  if (p.silu) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) dy[v] *= d[v];
  }
}

// weight and bias of VEC channels from c on (both arrays may start anywhere)
template <int VEC>
__device__ __forceinline__ void load_params(const NormParams& p, long long c, float (&w)[VEC], float (&b)[VEC]) {
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    w[v] = p.w != nullptr ? p.w[c + v] : 1.0f;
    b[v] = p.b != nullptr ? p.b[c + v] : 0.0f;
  }
}

// Sums of (a, b) per thread over the CTA's warps, in warp order, written by warp 0.
template <int VEC>
__device__ __forceinline__ void write_partials(float* part, long long row, long long C, long long c, bool live,
                                               const float (&a)[VEC], const float (&b)[VEC]) {
  __shared__ float red[kWarps][32][2 * VEC + 1];
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    red[threadIdx.y][threadIdx.x][v] = a[v];
    red[threadIdx.y][threadIdx.x][VEC + v] = b[v];
  }
  __syncthreads();
  if (!live) return;
  for (int j = threadIdx.y; j < 2 * VEC; j += kWarps) {
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += red[w][threadIdx.x][j];
    part[(row * 2 + (j >= VEC)) * C + c + j % VEC] = s;
  }
}

// Rows ahead of the one in work: kDepth rows of every tensor, copied asynchronously into slots of shared memory
// that only the thread itself reads, so no barrier is needed and depth costs no registers.  (A prefetch of one
// row in registers kept 22 KB per SM in flight and reached half the bandwidth.)
template <typename T, int VEC, int K, int TENSORS>
struct Slots {
  using Vec = ssm::Raw<T, VEC>;
  static constexpr int kRow = TENSORS * K * 32 * kWarps * (int)sizeof(Vec);
  static constexpr int kDepth = kRow * 4 <= 48 * 1024 ? 4 : 2;
  static constexpr size_t kBytes = (size_t)kDepth * kRow;
  Vec* slots;
  int tid;
  __device__ Slots(unsigned char* smem) : slots(reinterpret_cast<Vec*>(smem)), tid(threadIdx.y * 32 + threadIdx.x) {}
  __device__ Vec* slot(int stage, int tensor, int i = 0) { return slots + ((stage * TENSORS + tensor) * K + i) * 32 * kWarps + tid; }
  // src may be anything readable where ok is false: the slot becomes zero
  __device__ void copy(Vec* dst, const void* src, bool ok) {
    if constexpr (sizeof(Vec) >= 4) {
      asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(ssm::smem_u32(dst)), "l"(src),
                   "n"((int)sizeof(Vec)), "r"(ok ? (int)sizeof(Vec) : 0)
                   : "memory");
    } else {
      if (ok) dst->load(static_cast<const T*>(src));
      else dst->zero();
    }
  }
  __device__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
  __device__ void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory"); }
  __device__ void drain() { asm volatile("cp.async.wait_all;" ::: "memory"); }   // before the kernel ends
};

// ---- one position per sample ----------------------------------------------------------------
// WPG = 1: lpg lanes (a power of two) share a group, the CTA's warps take different rows; blockIdx.y
// selects 32 / lpg groups.  WPG = kWarps: the CTA shares one group, blockIdx.y selects it.
// Vector i of a lane starts at channel (lane + i lpg) VEC of the group.
template <int WPG>
struct Place {
  int lane;          // within the group
  int lpg;
  long long c0;      // first channel of the group
  bool live;         // the group exists
  long long row, step;
  __device__ Place(const NormParams& p, int lpg_) {
    long long group;
    if (WPG == 1) {
      lpg = lpg_;
      lane = threadIdx.x & (lpg - 1);
      group = (long long)blockIdx.y * (32 / lpg) + threadIdx.x / lpg;
      row = (long long)blockIdx.x * kWarps + threadIdx.y;
      step = (long long)gridDim.x * kWarps;
    } else {
      lpg = 32 * WPG;
      lane = threadIdx.y * 32 + threadIdx.x;
      group = blockIdx.y;
      row = blockIdx.x;
      step = gridDim.x;
    }
    live = group < p.G;
    c0 = group * p.cg;
  }
};
template <int WPG>
__device__ __forceinline__ float group_sum(float x, int lpg) {
  if (WPG == 1) {
    for (int m = lpg >> 1; m >= 1; m >>= 1) x += __shfl_xor_sync(0xffffffffu, x, m);
    return x;
  }
  __shared__ float red[kWarps];
  x = ssm::group_allreduce<32, 1>(x);
  __syncthreads();
  if (threadIdx.x == 0) red[threadIdx.y] = x;
  __syncthreads();
  float s = 0.0f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) s += red[w];
  return s;
}

// Mean (of the centred form) and rstd of the group whose lane holds x (zero past the group's end);
// x becomes x - mean.
template <int WPG, int VEC, int K>
__device__ __forceinline__ float row_stats(const NormParams& p, const Place<WPG>& at, float (&x)[K][VEC]) {
  const float inv = 1.0f / (float)p.cg;
  if (p.center) {
    float mean = 0.0f;
#pragma unroll
    for (int i = 0; i < K; ++i)
#pragma unroll
      for (int v = 0; v < VEC; ++v) mean += x[i][v];
    mean = group_sum<WPG>(mean, at.lpg) * inv;
#pragma unroll
    for (int i = 0; i < K; ++i)
      if ((at.lane + i * at.lpg) * VEC < p.cg) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) x[i][v] -= mean;
      }
  }
  float q = 0.0f;
#pragma unroll
  for (int i = 0; i < K; ++i)
#pragma unroll
    for (int v = 0; v < VEC; ++v) q = fmaf(x[i][v], x[i][v], q);
  return rsqrtf(fmaf(group_sum<WPG>(q, at.lpg), inv, p.eps));
}

template <typename T, int VEC, int K, bool BWD>
struct RowQueue : Slots<T, VEC, K, BWD ? 3 : 2> {
  using Base = Slots<T, VEC, K, BWD ? 3 : 2>;
  using Base::Base;
  template <int WPG>
  __device__ void fetch(const NormParams& p, const Place<WPG>& at, long long r, int stage) {
#pragma unroll
    for (int i = 0; i < K; ++i) {
      const int c = (at.lane + i * at.lpg) * VEC;
      const bool ok = at.live && r < p.N && c < p.cg;
      const long long rr = ok ? r : 0, cc = ok ? at.c0 + c : 0;
      this->copy(this->slot(stage, 0, i), static_cast<const T*>(p.x) + rr * p.xs + cc, ok);
      if (p.gate) this->copy(this->slot(stage, 1, i), static_cast<const T*>(p.z) + rr * p.zs + cc, ok);
      if (BWD) this->copy(this->slot(stage, 2, i), static_cast<const T*>(p.dy) + rr * p.gs + cc, ok);
    }
    this->commit();
  }
};

// The number of rows is the same for all of a CTA's warps, so that group_sum's barriers match; rows past
// the end work on zeros, and what comes of that (NaN where eps is 0) goes nowhere.  16384 x 5120 bf16 in 40 groups with a gate: 89 us, 5.6 TB/s of the tensors' bytes; issue
// slots are 78 % taken (13 operations an element, 16 of every 32 elements' special functions).
template <typename T, int VEC, int K, int WPG>
__global__ void __launch_bounds__(32 * kWarps) norm_rows_fwd(const __grid_constant__ NormParams p, int lpg) {
  extern __shared__ __align__(16) unsigned char smem[];
  const Place<WPG> at(p, lpg);
  RowQueue<T, VEC, K, false> queue(smem);
#pragma unroll
  for (int d = 0; d < queue.kDepth; ++d) queue.fetch(p, at, at.row + d * at.step, d);
  float w[K][VEC], b[K][VEC];
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const int c = (at.lane + i * at.lpg) * VEC;
    if (at.live && c < p.cg) load_params<VEC>(p, at.c0 + c, w[i], b[i]);
  }
  int stage = 0;
  for (long long r0 = 0; r0 < p.N; r0 += at.step) {
    const long long r = r0 + at.row;
    if (WPG > 1 && r >= p.N) break;
    float x[K][VEC], z[K][VEC];
    queue.wait();
#pragma unroll
    for (int i = 0; i < K; ++i) {
      queue.slot(stage, 0, i)->widen(x[i]);
      if (p.gate) queue.slot(stage, 1, i)->widen(z[i]);
    }
    queue.fetch(p, at, r + queue.kDepth * at.step, stage);
    stage = stage + 1 == queue.kDepth ? 0 : stage + 1;
    const float rstd = row_stats<WPG, VEC, K>(p, at, x);
#pragma unroll
    for (int i = 0; i < K; ++i) {
      const int c = (at.lane + i * at.lpg) * VEC;
      if (at.live && r < p.N && c < p.cg) {
        float o[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) x[i][v] *= rstd;
        norm_out(p, x[i], w[i], b[i], z[i], o);
        vec_store<T, VEC>(static_cast<T*>(p.y) + r * p.ys + at.c0 + c, o);
      }
    }
  }
  queue.drain();
}

// Parameter gradients stay in registers over a CTA's rows; WPG = 1 adds its warps' at the end.  The same tensors:
// 171 us, 4.9 TB/s; 112 registers leave 16 warps to an SM, 70 % of the issue slots taken.
template <typename T, int VEC, int K, int WPG>
__global__ void __launch_bounds__(32 * kWarps) norm_rows_bwd(const __grid_constant__ NormParams p, int lpg) {
  extern __shared__ __align__(16) unsigned char smem[];
  const Place<WPG> at(p, lpg);
  RowQueue<T, VEC, K, true> queue(smem);
#pragma unroll
  for (int d = 0; d < queue.kDepth; ++d) queue.fetch(p, at, at.row + d * at.step, d);
  const float inv = 1.0f / (float)p.cg;
  float dw[K][VEC], db[K][VEC], w[K][VEC], b[K][VEC];
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const int c = (at.lane + i * at.lpg) * VEC;
#pragma unroll
    for (int v = 0; v < VEC; ++v) dw[i][v] = db[i][v] = w[i][v] = b[i][v] = 0.0f;
    if (at.live && c < p.cg) load_params<VEC>(p, at.c0 + c, w[i], b[i]);
  }
  int stage = 0;
  for (long long r0 = 0; r0 < p.N; r0 += at.step) {
    const long long r = r0 + at.row;
    if (WPG > 1 && r >= p.N) break;
    const bool ok = at.live && r < p.N;
    float x[K][VEC], z[K][VEC], g[K][VEC];
    queue.wait();
#pragma unroll
    for (int i = 0; i < K; ++i) {
      queue.slot(stage, 0, i)->widen(x[i]);
      if (p.gate) queue.slot(stage, 1, i)->widen(z[i]);
      queue.slot(stage, 2, i)->widen(g[i]);
    }
    queue.fetch(p, at, r + queue.kDepth * at.step, stage);
    stage = stage + 1 == queue.kDepth ? 0 : stage + 1;
    const float rstd = row_stats<WPG, VEC, K>(p, at, x);
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < K; ++i) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) x[i][v] *= rstd;
      norm_grad(p, x[i], w[i], b[i], z[i], g[i]);
      if (ok) {                          // a row past the end is not a zero to the sums: with eps = 0 it is NaN
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          dw[i][v] = fmaf(g[i][v], x[i][v], dw[i][v]);
          db[i][v] += g[i][v];
        }
      }
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        g[i][v] *= w[i][v];
        s1 += g[i][v];
        s2 = fmaf(g[i][v], x[i][v], s2);
      }
    }
    s1 = p.center ? group_sum<WPG>(s1, at.lpg) * inv : 0.0f;
    s2 = group_sum<WPG>(s2, at.lpg) * inv;
#pragma unroll
    for (int i = 0; i < K; ++i) {
      const int c = (at.lane + i * at.lpg) * VEC;
      if (ok && c < p.cg) {
        float o[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) o[v] = rstd * (g[i][v] - fmaf(x[i][v], s2, s1));
        vec_store<T, VEC>(static_cast<T*>(p.dx) + r * p.dxs + at.c0 + c, o);
        if (p.gate) vec_store<T, VEC>(static_cast<T*>(p.dz) + r * p.dzs + at.c0 + c, z[i]);
      }
    }
  }
  queue.drain();
  float* part = p.part + (long long)blockIdx.x * 2 * p.C + at.c0;
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const int c = (at.lane + i * at.lpg) * VEC;
    const bool ok = at.live && c < p.cg;
    if (WPG == 1) {
      __shared__ float red[kWarps][32][2 * VEC + 1];
      __syncthreads();
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        red[threadIdx.y][threadIdx.x][v] = dw[i][v];
        red[threadIdx.y][threadIdx.x][VEC + v] = db[i][v];
      }
      __syncthreads();
      for (int j = threadIdx.y; j < 2 * VEC; j += kWarps) {
        float s = 0.0f;
#pragma unroll
        for (int q = 0; q < kWarps; ++q) s += red[q][threadIdx.x][j];
        if (ok) part[(j >= VEC ? p.C : 0) + c + j % VEC] = s;
      }
    } else if (ok) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        part[c + v] = dw[i][v];
        part[p.C + c + v] = db[i][v];
      }
    }
  }
}

// ---- one position per sample, groups too wide for registers: a warp per (sample, group) ------
template <typename T, bool BWD>
__global__ void __launch_bounds__(256) norm_group_sums(const __grid_constant__ NormParams p) {
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (i >= p.N * p.G) return;
  const long long n = i / p.G;
  const long long c0 = (i % p.G) * p.cg;
  const T* x = static_cast<const T*>(p.x) + n * p.xs + c0;
  const float inv = 1.0f / (float)p.cg;
  if constexpr (!BWD) {
    float mean = 0.0f, q = 0.0f;
    if (p.center) {
      for (int j = lane; j < p.cg; j += 32) mean += ssm::to_f32(x[j]);
      mean = ssm::group_allreduce<32, 1>(mean) * inv;
    }
    for (int j = lane; j < p.cg; j += 32) {
      const float d = ssm::to_f32(x[j]) - mean;
      q = fmaf(d, d, q);
    }
    q = ssm::group_allreduce<32, 1>(q);
    if (lane == 0) *reinterpret_cast<float2*>(p.stats + i * 2) = make_float2(mean, rsqrtf(fmaf(q, inv, p.eps)));
  } else {
    const T* dy = static_cast<const T*>(p.dy) + n * p.gs + c0;
    const T* z = static_cast<const T*>(p.z) + (p.gate ? n * p.zs + c0 : 0);
    const float2 st = *reinterpret_cast<const float2*>(p.stats + i * 2);
    float s1 = 0.0f, s2 = 0.0f;
    for (int j = lane; j < p.cg; j += 32) {
      float w[1], b[1], e[1] = {ssm::to_f32(dy[j])}, zj[1] = {p.gate ? ssm::to_f32(z[j]) : 0.0f};
      load_params<1>(p, c0 + j, w, b);
      const float n1[1] = {(ssm::to_f32(x[j]) - st.x) * st.y};
      norm_grad(p, n1, w, b, zj, e);
      e[0] *= w[0];
      s1 += e[0];
      s2 = fmaf(e[0], n1[0], s2);
    }
    s1 = ssm::group_allreduce<32, 1>(s1);
    s2 = ssm::group_allreduce<32, 1>(s2);
    if (lane == 0) *reinterpret_cast<float2*>(p.sums + i * 2) = make_float2(p.center ? s1 * inv : 0.0f, s2 * inv);
  }
}

// ---- element-wise and per-channel passes ----------------------------------------------------
// blockIdx.x = sample * nslab + slab (ROWS: one slab of the N samples' single rows).
struct Rows {
  long long n, r0, r1;
};
template <bool ROWS>
__device__ __forceinline__ Rows rows_of(const NormParams& p) {
  Rows s;
  const long long q = ROWS ? (long long)blockIdx.x : blockIdx.x % p.nslab;
  s.n = ROWS ? 0 : blockIdx.x / p.nslab;
  s.r0 = q * p.slab;
  const long long end = ROWS ? p.N : p.P;
  s.r1 = s.r0 + p.slab < end ? s.r0 + p.slab : end;
  return s;
}
template <bool ROWS>
__device__ __forceinline__ long long row_at(long long n, long long r, long long ss, long long ps) {
  return ROWS ? r * ss : n * ss + r * ps;
}

// A thread's rows of a slab, kWarps apart, in order: x, and where wanted dy and z.
template <typename T, int VEC, bool ROWS, bool GRAD>
struct SlabQueue : Slots<T, VEC, 1, GRAD ? 3 : 2> {
  using Base = Slots<T, VEC, 1, GRAD ? 3 : 2>;
  __device__ SlabQueue(unsigned char* smem) : Base(smem) {}
  __device__ void fetch(const NormParams& p, const Rows& s, long long c, long long r, bool z, int stage) {
    const bool ok = r < s.r1;
    const long long rr = ok ? r : s.r0;
    this->copy(this->slot(stage, 0), static_cast<const T*>(p.x) + row_at<ROWS>(s.n, rr, p.xs, p.xp) + c, ok);
    if (z) this->copy(this->slot(stage, 1), static_cast<const T*>(p.z) + row_at<ROWS>(s.n, rr, p.zs, p.zp) + c, ok);
    if (GRAD) this->copy(this->slot(stage, 2), static_cast<const T*>(p.dy) + row_at<ROWS>(s.n, rr, p.gs, p.gp) + c, ok);
    this->commit();
  }
  // f(row, x, z, dy) for every row
  template <typename F>
  __device__ void each(const NormParams& p, const Rows& s, long long c, bool gate, F f) {
#pragma unroll
    for (int d = 0; d < Base::kDepth; ++d) fetch(p, s, c, s.r0 + threadIdx.y + d * kWarps, gate, d);
    int stage = 0;
    for (long long r = s.r0 + threadIdx.y; r < s.r1; r += kWarps) {
      float x[VEC], z[VEC] = {}, g[VEC] = {};
      this->wait();
      this->slot(stage, 0)->widen(x);
      if (gate) this->slot(stage, 1)->widen(z);
      if (GRAD) this->slot(stage, 2)->widen(g);
      fetch(p, s, c, r + Base::kDepth * kWarps, gate, stage);
      stage = stage + 1 == Base::kDepth ? 0 : stage + 1;
      f(r, x, z, g);
    }
    this->drain();
  }
};

// The passes over a slab (8 x 8192 x 512 bf16: statistics 16 us, apply 29 us; x is read twice, 67 MB each time) are
// bound by memory.  Per (sample, slab, channel): mean and sum of squared deviations of the slab's rows, summed about the
// slab's first row so that a large common offset costs no digits; not centred, 0 and the sum of squares (about 0 that is
// infinite and not NaN where an element is infinite).
template <typename T, int VEC>
__global__ void __launch_bounds__(32 * kWarps) norm_col_stats(const __grid_constant__ NormParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  const long long c = ((long long)blockIdx.y * 32 + threadIdx.x) * VEC;
  const bool live = c < p.C;
  const Rows s = rows_of<false>(p);
  const T* x = static_cast<const T*>(p.x) + s.n * p.xs + c;
  float k[VEC], a[VEC], q[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) k[v] = a[v] = q[v] = 0.0f;
  if (live) {
    if (p.center) vec_load<T, VEC>(x + s.r0 * p.xp, k);
    SlabQueue<T, VEC, false, false>(smem).each(p, s, c, false, [&](long long, float (&t)[VEC], float (&)[VEC], float (&)[VEC]) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const float d = t[v] - k[v];
        a[v] += d;
        q[v] = fmaf(d, d, q[v]);
      }
    });
  }
  __shared__ float red[kWarps][32][2 * VEC + 1];
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    red[threadIdx.y][threadIdx.x][v] = a[v];
    red[threadIdx.y][threadIdx.x][VEC + v] = q[v];
  }
  __syncthreads();
  if (live && threadIdx.y == 0) {
    const float inv = 1.0f / (float)(s.r1 - s.r0);
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      float sa = 0.0f, sq = 0.0f;
      for (int w = 0; w < kWarps; ++w) {
        sa += red[w][threadIdx.x][v];
        sq += red[w][threadIdx.x][VEC + v];
      }
      float* o = p.part + ((long long)blockIdx.x * 2) * p.C + c + v;
      o[0] = p.center ? fmaf(sa, inv, k[v]) : 0.0f;
      o[p.C] = p.center ? fmaxf(sq - sa * sa * inv, 0.0f) : sq;
    }
  }
}

// Sum of a double over a CTA of 256 threads, in a fixed order, to all of them.
__device__ __forceinline__ double cta_sum(double x) {
  __shared__ double red[8];
  for (int k = 16; k >= 1; k >>= 1) x += __shfl_xor_sync(0xffffffffu, x, k);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
  __syncthreads();
  return ((red[0] + red[1]) + (red[2] + red[3])) + ((red[4] + red[5]) + (red[6] + red[7]));
}
// f(slab, channel of the group) for this thread's share of a sample's slabs x a group's channels.
template <typename F>
__device__ __forceinline__ void for_cells(const NormParams& p, F f) {
  const int cells = p.nslab * p.cg;
#pragma unroll 4
  for (int e = threadIdx.x; e < cells; e += 256) f(e / p.cg, e % p.cg);
}

// A CTA per (sample, group), or several in turn where there are more of them than a grid holds: mean and rstd from the
// slabs' per-channel means and squared deviations.
__global__ void __launch_bounds__(256) norm_combine_stats(const __grid_constant__ NormParams p) {
  const double m = (double)p.P * p.cg;
  auto rows = [&](int slab) {
    const long long r0 = slab * p.slab;
    return (double)((r0 + p.slab < p.P ? r0 + p.slab : p.P) - r0);
  };
  for (long long i = blockIdx.x; i < p.N * p.G; i += gridDim.x) {
    const float* part = p.part + i / p.G * p.nslab * 2 * p.C + i % p.G * p.cg;
    double mean = 0.0, q = 0.0;
    if (p.center) {
      for_cells(p, [&](int slab, int c) { mean += rows(slab) * part[(long long)slab * 2 * p.C + c]; });
      mean = cta_sum(mean) / m;
    }
    for_cells(p, [&](int slab, int c) {
      const float* at = part + (long long)slab * 2 * p.C + c;
      const double d = at[0] - mean;
      q += at[p.C] + rows(slab) * d * d;
    });
    q = cta_sum(q);
    if (threadIdx.x == 0)
      *reinterpret_cast<float2*>(p.stats + i * 2) = make_float2((float)mean, (float)(1.0 / sqrt(q / m + (double)p.eps)));
  }
}

template <typename T, int VEC, bool ROWS>
__global__ void __launch_bounds__(32 * kWarps) norm_apply_fwd(const __grid_constant__ NormParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  const long long c = ((long long)blockIdx.y * 32 + threadIdx.x) * VEC;
  if (c >= p.C) return;
  const Rows s = rows_of<ROWS>(p);
  float w[VEC], b[VEC], mean[VEC], rstd[VEC];
  load_params<VEC>(p, c, w, b);
  auto stats = [&](long long n) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      const float2 st = *reinterpret_cast<const float2*>(p.stats + (n * p.G + (c + v) / p.cg) * 2);
      mean[v] = st.x;
      rstd[v] = st.y;
    }
  };
  if (!ROWS) stats(s.n);
  SlabQueue<T, VEC, ROWS, false>(smem).each(p, s, c, p.gate, [&](long long r, float (&x)[VEC], float (&z)[VEC], float (&)[VEC]) {
    if (ROWS) stats(r);
    float o[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) x[v] = (x[v] - mean[v]) * rstd[v];
    norm_out(p, x, w, b, z, o);
    vec_store<T, VEC>(static_cast<T*>(p.y) + row_at<ROWS>(s.n, r, p.ys, p.yp) + c, o);
  });
}

// Per (sample, slab, channel) (ROWS: per (slab, channel)): sums of e n and of e.
template <typename T, int VEC, bool ROWS>
__global__ void __launch_bounds__(32 * kWarps) norm_col_grads(const __grid_constant__ NormParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  const long long c = ((long long)blockIdx.y * 32 + threadIdx.x) * VEC;
  const bool live = c < p.C;
  const Rows s = rows_of<ROWS>(p);
  float w[VEC], b[VEC], mean[VEC], rstd[VEC], dw[VEC], db[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) dw[v] = db[v] = 0.0f;
  if (live) {
    load_params<VEC>(p, c, w, b);
    auto stats = [&](long long n) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const float2 st = *reinterpret_cast<const float2*>(p.stats + (n * p.G + (c + v) / p.cg) * 2);
        mean[v] = st.x;
        rstd[v] = st.y;
      }
    };
    if (!ROWS) stats(s.n);
    SlabQueue<T, VEC, ROWS, true>(smem).each(p, s, c, p.gate, [&](long long r, float (&x)[VEC], float (&z)[VEC], float (&g)[VEC]) {
      if (ROWS) stats(r);
#pragma unroll
      for (int v = 0; v < VEC; ++v) x[v] = (x[v] - mean[v]) * rstd[v];
      norm_grad(p, x, w, b, z, g);
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        dw[v] = fmaf(g[v], x[v], dw[v]);
        db[v] += g[v];
      }
    });
  }
  write_partials<VEC>(p.part, blockIdx.x, p.C, c, live, dw, db);
}

// s1 / M and s2 / M from the channels' sums; CTAs as in norm_combine_stats.
__global__ void __launch_bounds__(256) norm_combine_sums(const __grid_constant__ NormParams p) {
  const double m = (double)p.P * p.cg;
  for (long long i = blockIdx.x; i < p.N * p.G; i += gridDim.x) {
    const long long c0 = i % p.G * p.cg;
    const float* part = p.part + i / p.G * p.nslab * 2 * p.C + c0;
    double s1 = 0.0, s2 = 0.0;
    for_cells(p, [&](int slab, int c) {
      const float* at = part + (long long)slab * 2 * p.C + c;
      const double w = p.w != nullptr ? p.w[c0 + c] : 1.0f;
      s2 += w * at[0];
      s1 += w * at[p.C];
    });
    s2 = cta_sum(s2);
    s1 = cta_sum(s1);
    if (threadIdx.x == 0)
      *reinterpret_cast<float2*>(p.sums + i * 2) = make_float2(p.center ? (float)(s1 / m) : 0.0f, (float)(s2 / m));
  }
}

template <typename T, int VEC, bool ROWS>
__global__ void __launch_bounds__(32 * kWarps) norm_apply_bwd(const __grid_constant__ NormParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  const long long c = ((long long)blockIdx.y * 32 + threadIdx.x) * VEC;
  if (c >= p.C) return;
  const Rows s = rows_of<ROWS>(p);
  float w[VEC], b[VEC], mean[VEC], rstd[VEC], s1[VEC], s2[VEC];
  load_params<VEC>(p, c, w, b);
  auto stats = [&](long long n) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      const long long at = (n * p.G + (c + v) / p.cg) * 2;
      const float2 st = *reinterpret_cast<const float2*>(p.stats + at);
      const float2 su = *reinterpret_cast<const float2*>(p.sums + at);
      mean[v] = st.x;
      rstd[v] = st.y;
      s1[v] = su.x;
      s2[v] = su.y;
    }
  };
  if (!ROWS) stats(s.n);
  SlabQueue<T, VEC, ROWS, true>(smem).each(p, s, c, p.gate, [&](long long r, float (&x)[VEC], float (&z)[VEC], float (&g)[VEC]) {
    if (ROWS) stats(r);
    float o[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) x[v] = (x[v] - mean[v]) * rstd[v];
    norm_grad(p, x, w, b, z, g);
#pragma unroll
    for (int v = 0; v < VEC; ++v) o[v] = rstd[v] * (g[v] * w[v] - fmaf(x[v], s2[v], s1[v]));
    vec_store<T, VEC>(static_cast<T*>(p.dx) + row_at<ROWS>(s.n, r, p.dxs, p.dxp) + c, o);
    if (p.gate) vec_store<T, VEC>(static_cast<T*>(p.dz) + row_at<ROWS>(s.n, r, p.dzs, p.dzp) + c, z);
  });
}

// dw and db: the partial rows summed in a fixed order (a warp takes every kWarps-th row, the warps'
// sums are added in warp order), in fp64: there are as many as samples where these are short.
__global__ void __launch_bounds__(32 * kWarps) norm_param_grads(const __grid_constant__ NormParams p, long long nparts) {
  __shared__ double red[kWarps][32];
  const long long c = (long long)blockIdx.x * 32 + threadIdx.x;
  const int which = blockIdx.y;
  float* out = which ? p.db : p.dw;
  double s = 0.0;
  if (c < p.C) {
#pragma unroll 8
    for (long long q = threadIdx.y; q < nparts; q += kWarps) s += (double)p.part[(q * 2 + which) * p.C + c];
  }
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < p.C && out != nullptr) {
    double t = 0.0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) t += red[w][threadIdx.x];
    out[c] = (float)t;
  }
}

// ---- host -----------------------------------------------------------------------------------
int fail(int code, const char* fmt, long long a = 0, long long b = 0) {
  char msg[256];
  snprintf(msg, sizeof(msg), fmt, a, b);
  return ssm::report_error(code, msg);
}

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// Slabs of rows: `ctas` CTAs in all, at least 2 rows per warp in each, and at most kChain rows after one another, `side` of
// which are taken side by side.  Sized for fp32 vectors whatever the type, so that the workspace size needs no type.
void plan_slabs(long long ctas, long long units, long long rows, long long C, int side, int* nslab, long long* slab) {
  const long long col_tiles = ceil_div(C, 128);
  long long n = ceil_div(ctas, units * col_tiles);
  n = std::min(n, ceil_div(rows, 2 * kWarps));
  n = std::max<long long>({n, ceil_div(rows, side * kChain), 1});
  *slab = ceil_div(rows, n);
  *nslab = (int)ceil_div(rows, *slab);
}

size_t round256(size_t x) { return (x + 255) & ~size_t(255); }

// The widest vector (a power of two elements, at most 16 bytes) that divides cg channels and at which every row
// of every view starts aligned.
int rows_vec(int cg, int es, std::initializer_list<ssm_view> views) {
  int vec = 16 / es;
  while (cg % vec != 0) vec /= 2;
  for (const ssm_view& v : views) {
    if (v.ptr == nullptr) continue;
    while (vec > 1 && (reinterpret_cast<uintptr_t>(v.ptr) % (vec * es) != 0 || v.batch_stride % vec != 0 ||
                       v.row_stride % vec != 0))
      vec /= 2;
  }
  return vec;
}

int check_shape(int64_t N, int64_t P, int64_t C, int64_t G) {
  if (N < 1 || P < 1 || C < 1) return fail(SSM_ERR_INVALID, "group_norm: samples, positions and channels must be positive");
  if (G < 1 || C % G != 0) return fail(SSM_ERR_INVALID, "group_norm: %lld channels do not split into %lld groups", C, G);
  // 2^40 elements are more than a GPU holds; below that the grids over slabs of rows fit
  if (N > (1LL << 30) || P > (1LL << 30) || C > (1LL << 20) || N * C > (1LL << 40) || P > (1LL << 40) / (N * C))
    return fail(SSM_ERR_INVALID, "group_norm: shape out of range (samples %lld, channels %lld)", N, C);
  return SSM_OK;
}
int check_act(const char* what, const ssm_view& v, int dtype, bool required) {
  char msg[160];
  if (v.ptr == nullptr) {
    if (!required) return SSM_OK;
    snprintf(msg, sizeof(msg), "group_norm: %s is required", what);
    return ssm::report_error(SSM_ERR_INVALID, msg);
  }
  if (v.dtype != dtype) {
    snprintf(msg, sizeof(msg), "group_norm: %s must have x's dtype", what);
    return ssm::report_error(SSM_ERR_DTYPE, msg);
  }
  return SSM_OK;
}

// How the rows kernels share a group of cg channels in vectors of vec: lanes (0: eight warps), vectors
// per lane (a power of two, at most 32 channels in all); K = 0 where the group does not fit.
struct RowsForm {
  int lpg, k;
};
RowsForm rows_form(int cg, int vec) {
  const int nvec = cg / vec, most = std::min(8, 32 / vec);
  RowsForm f = {1, 1};
  while (f.lpg < 32 && f.lpg < nvec) f.lpg *= 2;
  while (f.k < most && f.lpg * f.k < nvec) f.k *= 2;
  if (f.lpg * f.k >= nvec) return f;
  f = {0, 1};
  if (32 * kWarps < nvec) f.k = most;
  if (32 * kWarps * f.k < nvec) f.k = 0;
  return f;
}

template <typename T, int VEC, int K, int WPG>
cudaError_t launch_rows(NormParams& p, bool bwd, int lpg, cudaStream_t st) {
  const dim3 block(32, kWarps);
  const int per = WPG == 1 ? 32 / lpg : 1;                         // groups per CTA
  const unsigned gy = (unsigned)ceil_div(p.G, per);
  // one wave: rows ahead are on their way while a CTA works, so more CTAs than fit only start the queue again
  const long long rows = WPG == 1 ? ceil_div(p.N, kWarps) : p.N;
  auto ctas = [&](int fit, long long most) {
    return std::max<long long>(1, std::min({rows, most, (long long)148 * std::max(fit, 1) / gy}));
  };
  if (bwd) {
    constexpr size_t smem = RowQueue<T, VEC, K, true>::kBytes;
    constexpr auto kern = norm_rows_bwd<T, VEC, K, WPG>;
    // as many waves as kChain asks for (the plan has room for that many partial rows)
    const long long one = ctas(ssm::ctas_per_sm<kern>(32 * kWarps, smem), p.nslab);
    p.nslab = (int)std::min<long long>(p.nslab, one * ceil_div(rows, one * kChain));
    kern<<<dim3((unsigned)p.nslab, gy), block, smem, st>>>(p, lpg);
  } else {
    constexpr size_t smem = RowQueue<T, VEC, K, false>::kBytes;
    constexpr auto kern = norm_rows_fwd<T, VEC, K, WPG>;
    kern<<<dim3((unsigned)ctas(ssm::ctas_per_sm<kern>(32 * kWarps, smem), rows), gy), block, smem, st>>>(p, lpg);
  }
  return cudaGetLastError();
}
template <typename T, int VEC>
cudaError_t run_rows(NormParams& p, bool bwd, RowsForm f, cudaStream_t st) {
  constexpr int kMost = 32 / VEC < 8 ? 32 / VEC : 8;
  if (f.lpg == 0) return f.k == 1 ? launch_rows<T, VEC, 1, kWarps>(p, bwd, 0, st) : launch_rows<T, VEC, kMost, kWarps>(p, bwd, 0, st);
  if (f.k == 1) return launch_rows<T, VEC, 1, 1>(p, bwd, f.lpg, st);
  if (f.k == 2) return launch_rows<T, VEC, 2, 1>(p, bwd, f.lpg, st);
  if (f.k == 4) return launch_rows<T, VEC, 4, 1>(p, bwd, f.lpg, st);
  if constexpr (kMost == 8) return launch_rows<T, VEC, 8, 1>(p, bwd, f.lpg, st);
  return cudaErrorInvalidValue;
}
// The widest vector that divides a group and every row start.
template <typename T>
cudaError_t run_rows_any(NormParams& p, bool bwd, int vec, RowsForm f, cudaStream_t st) {
  if constexpr (sizeof(T) == 2)
    if (vec == 8) return run_rows<T, 8>(p, bwd, f, st);
  if (vec == 4) return run_rows<T, 4>(p, bwd, f, st);
  if (vec == 2) return run_rows<T, 2>(p, bwd, f, st);
  return run_rows<T, 1>(p, bwd, f, st);
}

template <auto Kern, typename Queue>
void launch_slabs(dim3 grid, const NormParams& p, cudaStream_t st) {
  if (Queue::kBytes > 24 * 1024) ssm::ctas_per_sm<Kern>(32 * kWarps, Queue::kBytes);   // beside static shared memory
  Kern<<<grid, dim3(32, kWarps), Queue::kBytes, st>>>(p);
}

unsigned groups_grid(const NormParams& p) { return (unsigned)std::min<long long>(p.N * p.G, (1LL << 31) - 1); }

// mean and rstd of every (sample, group) into p.stats
template <typename T, int VEC>
void run_stats(const NormParams& p, cudaStream_t st) {
  if (p.P == 1) {
    norm_group_sums<T, false><<<(unsigned)ceil_div(p.N * p.G, 8), 256, 0, st>>>(p);
    return;
  }
  const dim3 grid((unsigned)(p.N * p.nslab), (unsigned)ceil_div(ceil_div(p.C, VEC), 32));
  launch_slabs<norm_col_stats<T, VEC>, Slots<T, VEC, 1, 2>>(grid, p, st);
  norm_combine_stats<<<groups_grid(p), 256, 0, st>>>(p);
}

template <typename T, int VEC>
cudaError_t run_fwd(NormParams& p, cudaStream_t st) {
  const unsigned cols = (unsigned)ceil_div(ceil_div(p.C, VEC), 32);
  run_stats<T, VEC>(p, st);
  if (p.P == 1) launch_slabs<norm_apply_fwd<T, VEC, true>, Slots<T, VEC, 1, 2>>(dim3((unsigned)p.nslab, cols), p, st);
  else launch_slabs<norm_apply_fwd<T, VEC, false>, Slots<T, VEC, 1, 2>>(dim3((unsigned)(p.N * p.nslab), cols), p, st);
  return cudaGetLastError();
}

template <typename T, int VEC>
cudaError_t run_bwd(NormParams& p, bool stats_given, cudaStream_t st) {
  const unsigned cols = (unsigned)ceil_div(ceil_div(p.C, VEC), 32);
  if (!stats_given) run_stats<T, VEC>(p, st);
  if (p.P == 1) {
    norm_group_sums<T, true><<<(unsigned)ceil_div(p.N * p.G, 8), 256, 0, st>>>(p);
    launch_slabs<norm_col_grads<T, VEC, true>, Slots<T, VEC, 1, 3>>(dim3((unsigned)p.nslab, cols), p, st);
    launch_slabs<norm_apply_bwd<T, VEC, true>, Slots<T, VEC, 1, 3>>(dim3((unsigned)p.nslab, cols), p, st);
  } else {
    const dim3 grid((unsigned)(p.N * p.nslab), cols);
    launch_slabs<norm_col_grads<T, VEC, false>, Slots<T, VEC, 1, 3>>(grid, p, st);
    norm_combine_sums<<<groups_grid(p), 256, 0, st>>>(p);
    launch_slabs<norm_apply_bwd<T, VEC, false>, Slots<T, VEC, 1, 3>>(grid, p, st);
  }
  return cudaGetLastError();
}

template <typename T>
cudaError_t run_slabs(NormParams& p, bool bwd, bool stats_given, int vec, cudaStream_t st) {
  if constexpr (sizeof(T) == 2)
    if (vec == 8) return bwd ? run_bwd<T, 8>(p, stats_given, st) : run_fwd<T, 8>(p, st);
  if (vec == 4) return bwd ? run_bwd<T, 4>(p, stats_given, st) : run_fwd<T, 4>(p, st);
  if (vec == 2) return bwd ? run_bwd<T, 2>(p, stats_given, st) : run_fwd<T, 2>(p, st);
  return bwd ? run_bwd<T, 1>(p, stats_given, st) : run_fwd<T, 1>(p, st);
}

// Fills the shape and the slabs; returns the number of partial rows (each 2 C floats).
long long plan(NormParams& p, int64_t N, int64_t P, int64_t C, int64_t G) {
  p.N = N;
  p.P = P;
  p.C = C;
  p.G = (int)G;
  p.cg = (int)(C / G);
  if (P == 1) {
    plan_slabs(148 * 6, 1, N, C, 1, &p.nslab, &p.slab);
    return p.nslab;
  }
  plan_slabs(148 * 8, N, P, C, kWarps, &p.nslab, &p.slab);
  return N * p.nslab;
}

}  // namespace

extern "C" {

int ssm_group_norm_workspace_size(int64_t N, int64_t P, int64_t C, int64_t G, int32_t backward, size_t* bytes) {
  if (bytes == nullptr) return fail(SSM_ERR_INVALID, "group_norm: bytes is NULL");
  int rc = check_shape(N, P, C, G);
  if (rc) return rc;
  NormParams p = {};
  const size_t part = round256((size_t)plan(p, N, P, C, G) * 2 * C * sizeof(float));
  const size_t groups = round256((size_t)N * G * 2 * sizeof(float));
  // the rows kernels need none forward and only partial sums backward; single channels always fit worst
  const bool rows = P == 1 && rows_form(p.cg, 1).k != 0;
  if (backward) *bytes = part + (rows ? 0 : 2 * groups) + 256;
  else *bytes = rows ? 0 : (P > 1 ? part : 0) + groups + 256;
  return SSM_OK;
}

static void set_inputs(NormParams& p, ssm_view x, const float* weight, const float* bias, int32_t center, int32_t silu,
                       ssm_view z) {
  p.x = x.ptr;
  p.xs = x.batch_stride;
  p.xp = x.row_stride;
  p.z = z.ptr;
  p.zs = z.batch_stride;
  p.zp = z.row_stride;
  p.w = weight;
  p.b = bias;
  p.center = center ? 1 : 0;
  p.silu = silu ? 1 : 0;
  p.gate = z.ptr != nullptr;
}

int ssm_group_norm_fwd(int64_t N, int64_t P, int64_t C, int64_t G, ssm_view x, const float* weight, const float* bias,
                       float eps, int32_t center, int32_t silu, ssm_view z, ssm_view y, float* stats, void* workspace,
                       size_t workspace_bytes, void* stream) {
  int rc = check_shape(N, P, C, G);
  if (rc) return rc;
  if (x.ptr == nullptr) return fail(SSM_ERR_INVALID, "group_norm: x is required");
  if (x.dtype != SSM_F32 && x.dtype != SSM_BF16) return fail(SSM_ERR_DTYPE, "group_norm: x dtype %lld unsupported", x.dtype);
  if ((rc = check_act("z", z, x.dtype, false))) return rc;
  if ((rc = check_act("y", y, x.dtype, true))) return rc;
  size_t need = 0;
  ssm_group_norm_workspace_size(N, P, C, G, 0, &need);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(SSM_ERR_WORKSPACE, "group_norm: workspace of %lld bytes required, %lld given", (long long)need,
                (long long)workspace_bytes);
  NormParams p = {};
  const long long parts = plan(p, N, P, C, G);
  set_inputs(p, x, weight, bias, center, silu, z);
  p.y = const_cast<void*>(y.ptr);
  p.ys = y.batch_stride;
  p.yp = y.row_stride;
  p.eps = eps;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int es = x.dtype == SSM_BF16 ? 2 : 4;
  cudaError_t e;
  const int rv = rows_vec(p.cg, es, {x, z, y});
  const RowsForm f = rows_form(p.cg, rv);
  if (P == 1 && f.k != 0) {
    e = es == 2 ? run_rows_any<__nv_bfloat16>(p, false, rv, f, st) : run_rows_any<float>(p, false, rv, f, st);
  } else {
    unsigned char* cur = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~uintptr_t(255));
    if (P > 1) {
      p.part = reinterpret_cast<float*>(cur);
      cur += round256((size_t)parts * 2 * C * sizeof(float));
    }
    p.stats = stats != nullptr ? stats : reinterpret_cast<float*>(cur);
    const int vec = rows_vec((int)C, es, {x, z, y});
    e = es == 2 ? run_slabs<__nv_bfloat16>(p, false, true, vec, st) : run_slabs<float>(p, false, true, vec, st);
  }
  if (e != cudaSuccess) return fail(SSM_ERR_CUDA, "group_norm forward launch failed (error %lld)", (long long)e);
  return SSM_OK;
}

int ssm_group_norm_bwd(int64_t N, int64_t P, int64_t C, int64_t G, ssm_view x, const float* weight, const float* bias,
                       float eps, int32_t center, int32_t silu, ssm_view z, const float* stats, ssm_view dy,
                       ssm_view dx, float* dweight, float* dbias, ssm_view dz, void* workspace, size_t workspace_bytes,
                       void* stream) {
  int rc = check_shape(N, P, C, G);
  if (rc) return rc;
  if (x.ptr == nullptr) return fail(SSM_ERR_INVALID, "group_norm: x is required");
  if (x.dtype != SSM_F32 && x.dtype != SSM_BF16) return fail(SSM_ERR_DTYPE, "group_norm: x dtype %lld unsupported", x.dtype);
  if ((rc = check_act("z", z, x.dtype, false))) return rc;
  if ((rc = check_act("dy", dy, x.dtype, true))) return rc;
  if ((rc = check_act("dx", dx, x.dtype, true))) return rc;
  if ((rc = check_act("dz", dz, x.dtype, z.ptr != nullptr))) return rc;
  size_t need = 0;
  ssm_group_norm_workspace_size(N, P, C, G, 1, &need);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(SSM_ERR_WORKSPACE, "group_norm: workspace of %lld bytes required, %lld given", (long long)need,
                (long long)workspace_bytes);
  NormParams p = {};
  const long long parts = plan(p, N, P, C, G);
  set_inputs(p, x, weight, bias, center, silu, z);
  p.eps = eps;
  p.dy = dy.ptr;
  p.gs = dy.batch_stride;
  p.gp = dy.row_stride;
  p.dx = const_cast<void*>(dx.ptr);
  p.dxs = dx.batch_stride;
  p.dxp = dx.row_stride;
  p.dz = const_cast<void*>(dz.ptr);
  p.dzs = dz.batch_stride;
  p.dzp = dz.row_stride;
  p.dw = dweight;
  p.db = dbias;
  unsigned char* cur = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~uintptr_t(255));
  p.part = reinterpret_cast<float*>(cur);
  cur += round256((size_t)parts * 2 * C * sizeof(float));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int es = x.dtype == SSM_BF16 ? 2 : 4;
  cudaError_t e;
  long long nparts = parts;
  const int rv = rows_vec(p.cg, es, {x, z, dy, dx, dz});
  const RowsForm f = rows_form(p.cg, rv);
  if (P == 1 && f.k != 0) {
    e = es == 2 ? run_rows_any<__nv_bfloat16>(p, true, rv, f, st) : run_rows_any<float>(p, true, rv, f, st);
    nparts = p.nslab;
  } else {
    p.sums = reinterpret_cast<float*>(cur);
    cur += round256((size_t)N * G * 2 * sizeof(float));
    p.stats = stats != nullptr ? const_cast<float*>(stats) : reinterpret_cast<float*>(cur);
    const int vec = rows_vec((int)C, es, {x, z, dy, dx, dz});
    const bool given = stats != nullptr;
    e = es == 2 ? run_slabs<__nv_bfloat16>(p, true, given, vec, st) : run_slabs<float>(p, true, given, vec, st);
  }
  if (e == cudaSuccess && (dweight != nullptr || dbias != nullptr)) {
    norm_param_grads<<<dim3((unsigned)ceil_div(C, 32), 2), dim3(32, kWarps), 0, st>>>(p, nparts);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) return fail(SSM_ERR_CUDA, "group_norm backward launch failed (error %lld)", (long long)e);
  return SSM_OK;
}

}  // extern "C"
