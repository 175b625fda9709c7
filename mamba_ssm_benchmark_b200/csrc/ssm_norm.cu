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
// A thread owns VEC consecutive channels (16 bytes where the layout allows, else one element); a warp
// reads 32 consecutive vectors of a row.  Memory bounds every form; which launch does what:
//   * one position, group = a power of two <= 32 vectors ("rows"): one kernel, every tensor moved
//     once; the group sums are butterflies over the group's lanes, mean and variance two passes over
//     registers.
//   * one position, any other group width: a warp per (sample, group) for the sums, then the same
//     element-wise kernels as below with a stride of one sample per row.
//   * more positions: per-(slab of rows, channel) partial sums, a combine per (sample, group), an
//     element-wise pass (the tensors are read twice).
// All sums are fp32 (the combines fp64) in a fixed order: no atomics, results are reproducible.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdio>

#include "ssm_b200.h"
#include "ssm_vec.cuh"

namespace ssm {
int report_error(int code, const char* msg);
}  // namespace ssm

namespace {

using ssm::vec_load;
using ssm::vec_store;

constexpr int kWarps = 8;           // warps per CTA: rows taken side by side
constexpr int kTargetCtas = 148 * 4;

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

// y from the normalised value
__device__ __forceinline__ float norm_out(const NormParams& p, float n, float w, float b, float z) {
  float a = fmaf(n, w, b);
  if (p.silu) a *= ssm::sigmoid(a);
  return p.gate ? a * (z * ssm::sigmoid(z)) : a;
}
// e = d loss / d (n w + b), and dz
__device__ __forceinline__ float norm_grad(const NormParams& p, float n, float w, float b, float z, float dy,
                                           float& dz) {
  const float pre = fmaf(n, w, b);
  float a = pre, e = dy;
  if (p.silu) {
    const float s = ssm::sigmoid(pre);
    a = pre * s;
    e *= dsilu(pre, s);
  }
  if (p.gate) {
    const float s = ssm::sigmoid(z);
    e *= z * s;
    dz = dy * a * dsilu(z, s);
  }
  return e;
}

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

// ---- one position per sample, group = lpg lanes --------------------------------------------
template <typename T, int VEC, int U>
__global__ void __launch_bounds__(32 * kWarps) norm_rows_fwd(const NormParams p, int lpg) {
  const long long c = ((long long)blockIdx.y * 32 + threadIdx.x) * VEC;
  const bool live = c < p.C;
  const float inv = 1.0f / (float)p.cg;
  float w[VEC], b[VEC];
  if (live) load_params<VEC>(p, c, w, b);
  const long long r0 = (long long)blockIdx.x * kWarps * U + threadIdx.y;
  float x[U][VEC], z[U][VEC];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long r = r0 + u * kWarps;
#pragma unroll
    for (int v = 0; v < VEC; ++v) x[u][v] = z[u][v] = 0.0f;
    if (live && r < p.N) {
      vec_load<T, VEC>(static_cast<const T*>(p.x) + r * p.xs + c, x[u]);
      if (p.gate) vec_load<T, VEC>(static_cast<const T*>(p.z) + r * p.zs + c, z[u]);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long r = r0 + u * kWarps;
    float mean = 0.0f, q = 0.0f;
    if (p.center) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) mean += x[u][v];
      for (int m = lpg >> 1; m >= 1; m >>= 1) mean += __shfl_xor_sync(0xffffffffu, mean, m);
      mean *= inv;
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      x[u][v] -= mean;
      q = fmaf(x[u][v], x[u][v], q);
    }
    for (int m = lpg >> 1; m >= 1; m >>= 1) q += __shfl_xor_sync(0xffffffffu, q, m);
    const float rstd = rsqrtf(fmaf(q, inv, p.eps));
    if (live && r < p.N) {
      float o[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) o[v] = norm_out(p, x[u][v] * rstd, w[v], b[v], z[u][v]);
      vec_store<T, VEC>(static_cast<T*>(p.y) + r * p.ys + c, o);
      if (p.stats != nullptr && threadIdx.x % lpg == 0)
        *reinterpret_cast<float2*>(p.stats + (r * p.G + c / p.cg) * 2) = make_float2(mean, rstd);
    }
  }
}

// Rows r = slab, slab + nslab, ... in steps of kWarps rows; parameter gradients stay in registers.
template <typename T, int VEC>
__global__ void __launch_bounds__(32 * kWarps) norm_rows_bwd(const NormParams p, int lpg) {
  const long long c = ((long long)blockIdx.y * 32 + threadIdx.x) * VEC;
  const bool live = c < p.C;
  const float inv = 1.0f / (float)p.cg;
  float w[VEC], b[VEC], dw[VEC], db[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) w[v] = b[v] = dw[v] = db[v] = 0.0f;
  if (live) load_params<VEC>(p, c, w, b);
  for (long long r = (long long)blockIdx.x * kWarps + threadIdx.y; r < p.N; r += (long long)p.nslab * kWarps) {
    float x[VEC], z[VEC], g[VEC], dz[VEC], n[VEC];
    float2 st = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int v = 0; v < VEC; ++v) x[v] = z[v] = g[v] = 0.0f;
    if (live) {
      vec_load<T, VEC>(static_cast<const T*>(p.x) + r * p.xs + c, x);
      vec_load<T, VEC>(static_cast<const T*>(p.dy) + r * p.gs + c, g);
      if (p.gate) vec_load<T, VEC>(static_cast<const T*>(p.z) + r * p.zs + c, z);
      st = *reinterpret_cast<const float2*>(p.stats + (r * p.G + c / p.cg) * 2);
    }
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      n[v] = (x[v] - st.x) * st.y;
      g[v] = norm_grad(p, n[v], w[v], b[v], z[v], g[v], dz[v]);
      dw[v] = fmaf(g[v], n[v], dw[v]);
      db[v] += g[v];
      g[v] *= w[v];
      s1 += g[v];
      s2 = fmaf(g[v], n[v], s2);
    }
    for (int m = lpg >> 1; m >= 1; m >>= 1) {
      if (p.center) s1 += __shfl_xor_sync(0xffffffffu, s1, m);
      s2 += __shfl_xor_sync(0xffffffffu, s2, m);
    }
    s1 = p.center ? s1 * inv : 0.0f;
    s2 *= inv;
    if (live) {
      float o[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) o[v] = st.y * (g[v] - fmaf(n[v], s2, s1));
      vec_store<T, VEC>(static_cast<T*>(p.dx) + r * p.dxs + c, o);
      if (p.gate) vec_store<T, VEC>(static_cast<T*>(p.dz) + r * p.dzs + c, dz);
    }
  }
  write_partials<VEC>(p.part, blockIdx.x, p.C, c, live, dw, db);
}

// ---- one position per sample, any group width: a warp per (sample, group) ------------------
template <typename T, bool BWD>
__global__ void __launch_bounds__(256) norm_group_sums(const NormParams p) {
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
      float w[1], b[1], dz;
      load_params<1>(p, c0 + j, w, b);
      const float nn = (ssm::to_f32(x[j]) - st.x) * st.y;
      const float e = norm_grad(p, nn, w[0], b[0], p.gate ? ssm::to_f32(z[j]) : 0.0f, ssm::to_f32(dy[j]), dz) * w[0];
      s1 += e;
      s2 = fmaf(e, nn, s2);
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

// Per (sample, slab, channel): mean and sum of squared deviations of the slab's rows, summed about the
// slab's first row so that a large common offset costs no digits.
template <typename T, int VEC>
__global__ void __launch_bounds__(32 * kWarps) norm_col_stats(const NormParams p) {
  const long long c = ((long long)blockIdx.y * 32 + threadIdx.x) * VEC;
  const bool live = c < p.C;
  const Rows s = rows_of<false>(p);
  const T* x = static_cast<const T*>(p.x) + s.n * p.xs + c;
  float k[VEC], a[VEC], q[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) k[v] = a[v] = q[v] = 0.0f;
  if (live) {
    vec_load<T, VEC>(x + s.r0 * p.xp, k);
#pragma unroll 4
    for (long long r = s.r0 + threadIdx.y; r < s.r1; r += kWarps) {
      float t[VEC];
      vec_load<T, VEC>(x + r * p.xp, t);
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const float d = t[v] - k[v];
        a[v] += d;
        q[v] = fmaf(d, d, q[v]);
      }
    }
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
      o[0] = fmaf(sa, inv, k[v]);
      o[p.C] = fmaxf(sq - sa * sa * inv, 0.0f);
    }
  }
}

// A warp per (sample, group): mean and rstd from the slabs' per-channel means and squared deviations.
__global__ void __launch_bounds__(256) norm_combine_stats(const NormParams p) {
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (i >= p.N * p.G) return;
  const long long n = i / p.G, c0 = (i % p.G) * p.cg;
  const long long cells = (long long)p.nslab * p.cg;
  const double m = (double)p.P * p.cg;
  double mean = 0.0, q = 0.0;
  auto at = [&](long long e) { return ((n * p.nslab + e / p.cg) * 2) * p.C + c0 + e % p.cg; };
  auto rows = [&](long long e) {
    const long long r0 = e / p.cg * p.slab;
    return (double)((r0 + p.slab < p.P ? r0 + p.slab : p.P) - r0);
  };
  if (p.center) {
    for (long long e = lane; e < cells; e += 32) mean += rows(e) * p.part[at(e)];
    for (int k = 16; k >= 1; k >>= 1) mean += __shfl_xor_sync(0xffffffffu, mean, k);
    mean /= m;
  }
  for (long long e = lane; e < cells; e += 32) {
    const double d = p.part[at(e)] - mean;
    q += p.part[at(e) + p.C] + rows(e) * d * d;
  }
  for (int k = 16; k >= 1; k >>= 1) q += __shfl_xor_sync(0xffffffffu, q, k);
  if (lane == 0)
    *reinterpret_cast<float2*>(p.stats + i * 2) = make_float2((float)mean, (float)(1.0 / sqrt(q / m + (double)p.eps)));
}

template <typename T, int VEC, bool ROWS>
__global__ void __launch_bounds__(32 * kWarps) norm_apply_fwd(const NormParams p) {
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
#pragma unroll 4
  for (long long r = s.r0 + threadIdx.y; r < s.r1; r += kWarps) {
    float x[VEC], z[VEC], o[VEC];
    vec_load<T, VEC>(static_cast<const T*>(p.x) + row_at<ROWS>(s.n, r, p.xs, p.xp) + c, x);
    if (p.gate) vec_load<T, VEC>(static_cast<const T*>(p.z) + row_at<ROWS>(s.n, r, p.zs, p.zp) + c, z);
    if (ROWS) stats(r);
#pragma unroll
    for (int v = 0; v < VEC; ++v) o[v] = norm_out(p, (x[v] - mean[v]) * rstd[v], w[v], b[v], p.gate ? z[v] : 0.0f);
    vec_store<T, VEC>(static_cast<T*>(p.y) + row_at<ROWS>(s.n, r, p.ys, p.yp) + c, o);
  }
}

// Per (sample, slab, channel) (ROWS: per (slab, channel)): sums of e n and of e.
template <typename T, int VEC, bool ROWS>
__global__ void __launch_bounds__(32 * kWarps) norm_col_grads(const NormParams p) {
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
#pragma unroll 2
    for (long long r = s.r0 + threadIdx.y; r < s.r1; r += kWarps) {
      float x[VEC], z[VEC], g[VEC], dz;
      vec_load<T, VEC>(static_cast<const T*>(p.x) + row_at<ROWS>(s.n, r, p.xs, p.xp) + c, x);
      vec_load<T, VEC>(static_cast<const T*>(p.dy) + row_at<ROWS>(s.n, r, p.gs, p.gp) + c, g);
      if (p.gate) vec_load<T, VEC>(static_cast<const T*>(p.z) + row_at<ROWS>(s.n, r, p.zs, p.zp) + c, z);
      if (ROWS) stats(r);
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const float n = (x[v] - mean[v]) * rstd[v];
        const float e = norm_grad(p, n, w[v], b[v], p.gate ? z[v] : 0.0f, g[v], dz);
        dw[v] = fmaf(e, n, dw[v]);
        db[v] += e;
      }
    }
  }
  write_partials<VEC>(p.part, blockIdx.x, p.C, c, live, dw, db);
}

// A warp per (sample, group): s1 / M and s2 / M from the channels' sums.
__global__ void __launch_bounds__(256) norm_combine_sums(const NormParams p) {
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (i >= p.N * p.G) return;
  const long long n = i / p.G, c0 = (i % p.G) * p.cg;
  const long long cells = (long long)p.nslab * p.cg;
  double s1 = 0.0, s2 = 0.0;
  for (long long e = lane; e < cells; e += 32) {
    const long long c = c0 + e % p.cg, o = ((n * p.nslab + e / p.cg) * 2) * p.C + c;
    const double w = p.w != nullptr ? p.w[c] : 1.0f;
    s2 += w * p.part[o];
    s1 += w * p.part[o + p.C];
  }
  for (int k = 16; k >= 1; k >>= 1) {
    s1 += __shfl_xor_sync(0xffffffffu, s1, k);
    s2 += __shfl_xor_sync(0xffffffffu, s2, k);
  }
  const double m = (double)p.P * p.cg;
  if (lane == 0)
    *reinterpret_cast<float2*>(p.sums + i * 2) = make_float2(p.center ? (float)(s1 / m) : 0.0f, (float)(s2 / m));
}

template <typename T, int VEC, bool ROWS>
__global__ void __launch_bounds__(32 * kWarps) norm_apply_bwd(const NormParams p) {
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
#pragma unroll 2
  for (long long r = s.r0 + threadIdx.y; r < s.r1; r += kWarps) {
    float x[VEC], z[VEC], g[VEC], dz[VEC], o[VEC];
    vec_load<T, VEC>(static_cast<const T*>(p.x) + row_at<ROWS>(s.n, r, p.xs, p.xp) + c, x);
    vec_load<T, VEC>(static_cast<const T*>(p.dy) + row_at<ROWS>(s.n, r, p.gs, p.gp) + c, g);
    if (p.gate) vec_load<T, VEC>(static_cast<const T*>(p.z) + row_at<ROWS>(s.n, r, p.zs, p.zp) + c, z);
    if (ROWS) stats(r);
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      const float n = (x[v] - mean[v]) * rstd[v];
      const float e = norm_grad(p, n, w[v], b[v], p.gate ? z[v] : 0.0f, g[v], dz[v]) * w[v];
      o[v] = rstd[v] * (e - fmaf(n, s2[v], s1[v]));
    }
    vec_store<T, VEC>(static_cast<T*>(p.dx) + row_at<ROWS>(s.n, r, p.dxs, p.dxp) + c, o);
    if (p.gate) vec_store<T, VEC>(static_cast<T*>(p.dz) + row_at<ROWS>(s.n, r, p.dzs, p.dzp) + c, dz);
  }
}

// dw and db: the partial rows summed in a fixed order (a warp takes every kWarps-th row, the warps'
// sums are added in warp order).
__global__ void __launch_bounds__(32 * kWarps) norm_param_grads(const NormParams p, long long nparts) {
  __shared__ float red[kWarps][32];
  const long long c = (long long)blockIdx.x * 32 + threadIdx.x;
  const int which = blockIdx.y;
  float* out = which ? p.db : p.dw;
  float s = 0.0f;
  if (c < p.C) {
#pragma unroll 4
    for (long long q = threadIdx.y; q < nparts; q += kWarps) s += p.part[(q * 2 + which) * p.C + c];
  }
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < p.C && out != nullptr) {
    float t = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) t += red[w][threadIdx.x];
    out[c] = t;
  }
}

// ---- host -----------------------------------------------------------------------------------
int fail(int code, const char* fmt, long long a = 0, long long b = 0) {
  char msg[256];
  snprintf(msg, sizeof(msg), fmt, a, b);
  return ssm::report_error(code, msg);
}

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// Slabs of rows: enough CTAs to fill the GPU a few times, at least 4 rows per warp in each.  Sized for
// 16-byte fp32 vectors whatever the type, so that the workspace size needs no type.
void plan_slabs(long long units, long long rows, long long C, int* nslab, long long* slab) {
  const long long col_tiles = ceil_div(C, 128);
  long long n = ceil_div(kTargetCtas, units * col_tiles);
  n = std::min(n, ceil_div(rows, 4 * kWarps));
  n = std::max<long long>(n, 1);
  *slab = ceil_div(rows, n);
  *nslab = (int)ceil_div(rows, *slab);
}

size_t round256(size_t x) { return (x + 255) & ~size_t(255); }

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool view_al(const ssm_view& v, int es) {
  return v.ptr == nullptr || (al16(v.ptr) && (v.batch_stride * es) % 16 == 0 && (v.row_stride * es) % 16 == 0);
}

int check_shape(int64_t N, int64_t P, int64_t C, int64_t G) {
  if (N < 1 || P < 1 || C < 1) return fail(SSM_ERR_INVALID, "group_norm: samples, positions and channels must be positive");
  if (G < 1 || C % G != 0) return fail(SSM_ERR_INVALID, "group_norm: %lld channels do not split into %lld groups", C, G);
  if (N > (1LL << 30) || P > (1LL << 30) || C > (1LL << 20))
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

// Lanes per group when the one-kernel rows form applies, else 0.
int rows_lanes(int64_t P, int cg, int vec) {
  if (P != 1 || cg % vec != 0) return 0;
  const int lanes = cg / vec;
  return lanes <= 32 && (lanes & (lanes - 1)) == 0 ? lanes : 0;
}

template <typename T, int VEC>
cudaError_t run_fwd(NormParams& p, cudaStream_t st) {
  const dim3 block(32, kWarps);
  const unsigned cols = (unsigned)ceil_div(ceil_div(p.C, VEC), 32);
  if (const int lpg = rows_lanes(p.P, p.cg, VEC)) {
    constexpr int U = 4;
    norm_rows_fwd<T, VEC, U><<<dim3((unsigned)ceil_div(p.N, kWarps * U), cols), block, 0, st>>>(p, lpg);
    return cudaGetLastError();
  }
  if (p.P == 1) {
    norm_group_sums<T, false><<<(unsigned)ceil_div(p.N * p.G, 8), 256, 0, st>>>(p);
    norm_apply_fwd<T, VEC, true><<<dim3((unsigned)p.nslab, cols), block, 0, st>>>(p);
    return cudaGetLastError();
  }
  const dim3 grid((unsigned)(p.N * p.nslab), cols);
  norm_col_stats<T, VEC><<<grid, block, 0, st>>>(p);
  norm_combine_stats<<<(unsigned)ceil_div(p.N * p.G, 8), 256, 0, st>>>(p);
  norm_apply_fwd<T, VEC, false><<<grid, block, 0, st>>>(p);
  return cudaGetLastError();
}

template <typename T, int VEC>
cudaError_t run_bwd(NormParams& p, cudaStream_t st) {
  const dim3 block(32, kWarps);
  const unsigned cols = (unsigned)ceil_div(ceil_div(p.C, VEC), 32);
  long long nparts = p.nslab;
  if (const int lpg = rows_lanes(p.P, p.cg, VEC)) {
    norm_rows_bwd<T, VEC><<<dim3((unsigned)p.nslab, cols), block, 0, st>>>(p, lpg);
  } else if (p.P == 1) {
    norm_group_sums<T, true><<<(unsigned)ceil_div(p.N * p.G, 8), 256, 0, st>>>(p);
    norm_col_grads<T, VEC, true><<<dim3((unsigned)p.nslab, cols), block, 0, st>>>(p);
    norm_apply_bwd<T, VEC, true><<<dim3((unsigned)p.nslab, cols), block, 0, st>>>(p);
  } else {
    nparts = p.N * p.nslab;
    const dim3 grid((unsigned)nparts, cols);
    norm_col_grads<T, VEC, false><<<grid, block, 0, st>>>(p);
    norm_combine_sums<<<(unsigned)ceil_div(p.N * p.G, 8), 256, 0, st>>>(p);
    norm_apply_bwd<T, VEC, false><<<grid, block, 0, st>>>(p);
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  if (p.dw != nullptr || p.db != nullptr) {
    norm_param_grads<<<dim3((unsigned)ceil_div(p.C, 32), 2), block, 0, st>>>(p, nparts);
    e = cudaGetLastError();
  }
  return e;
}

// Fills the shape and the slabs; returns the number of partial rows (each 2 C floats).
long long plan(NormParams& p, int64_t N, int64_t P, int64_t C, int64_t G) {
  p.N = N;
  p.P = P;
  p.C = C;
  p.G = (int)G;
  p.cg = (int)(C / G);
  if (P == 1) {
    plan_slabs(1, N, C, &p.nslab, &p.slab);
    return p.nslab;
  }
  plan_slabs(N, P, C, &p.nslab, &p.slab);
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
  if (backward) *bytes = part + groups + 256;
  else *bytes = (P > 1 ? part : 0) + groups + 256;
  return SSM_OK;
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
  if (workspace == nullptr || workspace_bytes < need)
    return fail(SSM_ERR_WORKSPACE, "group_norm: workspace of %lld bytes required, %lld given", (long long)need,
                (long long)workspace_bytes);
  NormParams p = {};
  const long long parts = plan(p, N, P, C, G);
  unsigned char* cur = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~uintptr_t(255));
  if (P > 1) {
    p.part = reinterpret_cast<float*>(cur);
    cur += round256((size_t)parts * 2 * C * sizeof(float));
  }
  p.stats = stats != nullptr ? stats : reinterpret_cast<float*>(cur);
  p.x = x.ptr;
  p.xs = x.batch_stride;
  p.xp = x.row_stride;
  p.z = z.ptr;
  p.zs = z.batch_stride;
  p.zp = z.row_stride;
  p.y = const_cast<void*>(y.ptr);
  p.ys = y.batch_stride;
  p.yp = y.row_stride;
  p.w = weight;
  p.b = bias;
  p.eps = eps;
  p.center = center ? 1 : 0;
  p.silu = silu ? 1 : 0;
  p.gate = z.ptr != nullptr;
  const int es = x.dtype == SSM_BF16 ? 2 : 4;
  const bool vec = C % (16 / es) == 0 && view_al(x, es) && view_al(z, es) && view_al(y, es);
  if (stats == nullptr && rows_lanes(P, p.cg, vec ? 16 / es : 1)) p.stats = nullptr;   // not needed, not written
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (x.dtype == SSM_BF16) e = vec ? run_fwd<__nv_bfloat16, 8>(p, st) : run_fwd<__nv_bfloat16, 1>(p, st);
  else e = vec ? run_fwd<float, 4>(p, st) : run_fwd<float, 1>(p, st);
  if (e != cudaSuccess) return fail(SSM_ERR_CUDA, "group_norm forward launch failed (error %lld)", (long long)e);
  return SSM_OK;
}

int ssm_group_norm_bwd(int64_t N, int64_t P, int64_t C, int64_t G, ssm_view x, const float* weight, const float* bias,
                       int32_t center, int32_t silu, ssm_view z, const float* stats, ssm_view dy, ssm_view dx,
                       float* dweight, float* dbias, ssm_view dz, void* workspace, size_t workspace_bytes,
                       void* stream) {
  int rc = check_shape(N, P, C, G);
  if (rc) return rc;
  if (x.ptr == nullptr || stats == nullptr) return fail(SSM_ERR_INVALID, "group_norm: x and stats are required");
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
  unsigned char* cur = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~uintptr_t(255));
  p.part = reinterpret_cast<float*>(cur);
  p.sums = reinterpret_cast<float*>(cur + round256((size_t)parts * 2 * C * sizeof(float)));
  p.stats = const_cast<float*>(stats);
  p.x = x.ptr;
  p.xs = x.batch_stride;
  p.xp = x.row_stride;
  p.z = z.ptr;
  p.zs = z.batch_stride;
  p.zp = z.row_stride;
  p.dy = dy.ptr;
  p.gs = dy.batch_stride;
  p.gp = dy.row_stride;
  p.dx = const_cast<void*>(dx.ptr);
  p.dxs = dx.batch_stride;
  p.dxp = dx.row_stride;
  p.dz = const_cast<void*>(dz.ptr);
  p.dzs = dz.batch_stride;
  p.dzp = dz.row_stride;
  p.w = weight;
  p.b = bias;
  p.dw = dweight;
  p.db = dbias;
  p.center = center ? 1 : 0;
  p.silu = silu ? 1 : 0;
  p.gate = z.ptr != nullptr;
  const int es = x.dtype == SSM_BF16 ? 2 : 4;
  const bool vec = C % (16 / es) == 0 && view_al(x, es) && view_al(z, es) && view_al(dy, es) && view_al(dx, es) &&
                   view_al(dz, es);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (x.dtype == SSM_BF16) e = vec ? run_bwd<__nv_bfloat16, 8>(p, st) : run_bwd<__nv_bfloat16, 1>(p, st);
  else e = vec ? run_bwd<float, 4>(p, st) : run_bwd<float, 1>(p, st);
  if (e != cudaSuccess) return fail(SSM_ERR_CUDA, "group_norm backward launch failed (error %lld)", (long long)e);
  return SSM_OK;
}

}  // extern "C"
