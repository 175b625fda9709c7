// ssm_rms_bwd.cu — backward of the root-mean-square norm with a residual (ssm_rms.cuh).
//
//   n = t rstd,  g = dy w:   d = dt + rstd (g - n mean(g n)),   dw = sum over rows of dy n
// d is the gradient of x and of the residual alike.  rstd comes from t again, which is read anyway.  The gradient of the weight
// stays in registers over a team's rows, at most kRmsChain of them; the teams of a CTA add theirs in order, and a second
// kernel adds the CTAs' partial rows in fp64: no atomics, results are reproducible.
#include <cstdio>
#include <initializer_list>

#include "ssm_b200.h"
#include "ssm_rms.cuh"

namespace ssm {
int report_error(int code, const char* msg);

namespace {

template <typename TX, typename TR, int VEC, int K>
__global__ void __launch_bounds__(kRmsThreads) rms_bwd(const __grid_constant__ RmsParams p, int wpr) {
  constexpr int kT = Slot<TR, VEC>::kBytes, kG = Slot<TX, VEC>::kBytes, kRow = K * (2 * kT + kG), kDepth = rms_depth(kRow);
  extern __shared__ __align__(16) unsigned char queue[];
  __shared__ float2 red[2 * kRmsThreads / 32];
  Team team(wpr, red);
  constexpr int nt = kRmsThreads;
  const int teams = nt / 32 / wpr;
  const long long step = (long long)gridDim.x * teams;
  long long row = (long long)blockIdx.x * teams + team.id;

  auto fetch = [&](long long r, int stage) {
    unsigned char* at = queue + (size_t)stage * kRow * nt;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (team.tid + k * team.size) * VEC;
      const bool ok = r < p.rows && c < p.C;
      Slot<TR, VEC>::fetch(at + (size_t)k * kT * nt, static_cast<const TR*>(p.t) + (ok ? r * p.ts + c : 0), ok);
      Slot<TX, VEC>::fetch(at + (size_t)(K * kT + k * kG) * nt, static_cast<const TX*>(p.y) + (ok ? r * p.ys + c : 0), ok);
      if (p.dt != nullptr)
        Slot<TR, VEC>::fetch(at + (size_t)(K * (kT + kG) + k * kT) * nt,
                             static_cast<const TR*>(p.dt) + (ok ? r * p.dts + c : 0), ok);
    }
    queue_commit();
  };
#pragma unroll
  for (int d = 0; d < kDepth; ++d) fetch(row + d * step, d);
  float w[K][VEC], dw[K][VEC];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (team.tid + k * team.size) * VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) w[k][i] = dw[k][i] = 0.0f;
    if (c < p.C) load_weight<VEC>(p, c, w[k]);
  }
  int stage = 0;
  for (; row < p.rows; row += step) {
    float t[K][VEC], g[K][VEC], d[K][VEC];
    float ss = 0.0f, gt = 0.0f;
    queue_wait<kDepth - 1>();
    const unsigned char* at = queue + (size_t)stage * kRow * nt;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      Slot<TR, VEC>::read(at + (size_t)k * kT * nt, t[k]);
      Slot<TX, VEC>::read(at + (size_t)(K * kT + k * kG) * nt, g[k]);
      if (p.dt != nullptr) {
        Slot<TR, VEC>::read(at + (size_t)(K * (kT + kG) + k * kT) * nt, d[k]);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) d[k][i] = 0.0f;
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        ss = fmaf(t[k][i], t[k][i], ss);
        gt = fmaf(g[k][i] * w[k][i], t[k][i], gt);
      }
    }
    fetch(row + kDepth * step, stage);
    stage = stage + 1 == kDepth ? 0 : stage + 1;
    const float2 s = team.sum(ss, gt);
    const float rstd = 1.0f / sqrtf(s.x * p.inv_c + p.eps);
    const float mean = s.y * rstd * p.inv_c;              // of g n
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (team.tid + k * team.size) * VEC;
      if (c >= p.C) continue;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float n = t[k][i] * rstd;
        dw[k][i] = fmaf(g[k][i], n, dw[k][i]);
        d[k][i] = fmaf(rstd, fmaf(-n, mean, g[k][i] * w[k][i]), d[k][i]);
      }
      write_piece<TX, VEC>(static_cast<TX*>(p.dx) + row * p.dxs + c, d[k]);
      if (p.dr != nullptr) write_piece<TR, VEC>(static_cast<TR*>(p.dr) + row * p.drs + c, d[k]);
    }
  }
  queue_wait<0>();
  if (p.part == nullptr) return;
  // the teams' gradients one after another through shared memory: thread j of every team has the same channels
  float* sum = reinterpret_cast<float*>(queue);           // [K * VEC][threads of a team]
  for (int q = 0; q < teams; ++q) {
    __syncthreads();
    if (team.id == q) {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          float& s = sum[(k * VEC + i) * team.size + team.tid];
          s = q == 0 ? dw[k][i] : s + dw[k][i];
        }
    }
  }
  if (team.id == teams - 1) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (team.tid + k * team.size) * VEC;
      if (c >= p.C) continue;
#pragma unroll
      for (int i = 0; i < VEC; ++i) p.part[(size_t)blockIdx.x * p.C + c + i] = sum[(k * VEC + i) * team.size + team.tid];
    }
  }
}

// Rows that no team holds: a CTA per row for the sums and d; rstd goes to `stat`.
template <typename TX, typename TR>
__global__ void __launch_bounds__(512) rms_bwd_long(const __grid_constant__ RmsParams p, float* stat) {
  __shared__ float2 red[2 * 16];
  Team team(16, red);
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const TR* t = static_cast<const TR*>(p.t) + row * p.ts;
    const TX* dy = static_cast<const TX*>(p.y) + row * p.ys;
    float ss = 0.0f, gt = 0.0f, w[1];
    for (int c = threadIdx.x; c < p.C; c += 512) {
      load_weight<1>(p, c, w);
      const float v = to_f32(t[c]);
      ss = fmaf(v, v, ss);
      gt = fmaf(to_f32(dy[c]) * w[0], v, gt);
    }
    const float2 s = team.sum(ss, gt);
    const float rstd = 1.0f / sqrtf(s.x * p.inv_c + p.eps), mean = s.y * rstd * p.inv_c;
    if (threadIdx.x == 0) stat[row] = rstd;
    for (int c = threadIdx.x; c < p.C; c += 512) {
      load_weight<1>(p, c, w);
      const float d0 = p.dt != nullptr ? to_f32(static_cast<const TR*>(p.dt)[row * p.dts + c]) : 0.0f;
      const float d = fmaf(rstd, fmaf(-to_f32(t[c]) * rstd, mean, to_f32(dy[c]) * w[0]), d0);
      static_cast<TX*>(p.dx)[row * p.dxs + c] = from_f32<TX>(d);
      if (p.dr != nullptr) static_cast<TR*>(p.dr)[row * p.drs + c] = from_f32<TR>(d);
    }
  }
}
// Their gradient of the weight: 32 channels and kRmsChain rows to a CTA, eight rows side by side.
template <typename TX, typename TR>
__global__ void __launch_bounds__(256) rms_bwd_cols(const __grid_constant__ RmsParams p, const float* stat) {
  __shared__ float red[8][32];
  const long long c = (long long)blockIdx.x * 32 + threadIdx.x;
  for (long long slab = blockIdx.y; slab * kRmsChain < p.rows; slab += gridDim.y) {
    const long long end = min(p.rows, (slab + 1) * kRmsChain);
    float s = 0.0f;
    if (c < p.C)
      for (long long r = slab * kRmsChain + threadIdx.y; r < end; r += 8)
        s = fmaf(to_f32(static_cast<const TX*>(p.y)[r * p.ys + c]), to_f32(static_cast<const TR*>(p.t)[r * p.ts + c]) * stat[r], s);
    red[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && c < p.C) {
      for (int i = 1; i < 8; ++i) s += red[i][threadIdx.x];
      p.part[slab * p.C + c] = s;
    }
    __syncthreads();
  }
}

// The partial rows in a fixed order: a warp takes every eighth, the warps' sums are added in order.
template <typename TW>
__global__ void __launch_bounds__(256) rms_dweight(const float* part, long long nparts, int C, TW* dw) {
  __shared__ double red[8][32];
  const long long c = (long long)blockIdx.x * 32 + threadIdx.x;
  double s = 0.0;
  if (c < C) {
#pragma unroll 8
    for (long long q = threadIdx.y; q < nparts; q += 8) s += (double)part[q * C + c];
  }
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < C) {
    for (int i = 1; i < 8; ++i) s += red[i][threadIdx.x];
    dw[c] = from_f32<TW>((float)s);
  }
}

// ---- host -----------------------------------------------------------------------------------
int fail(int code, const char* fmt, long long a = 0, long long b = 0) {
  char msg[256];
  snprintf(msg, sizeof(msg), fmt, a, b);
  return report_error(code, msg);
}

// Partial rows: a CTA each, of teams that take at most kRmsChain rows; or a slab of kRmsChain rows each.
constexpr long long kCtas = 148 * 8;
long long most_parts(long long rows) { return std::max(kCtas, rms_ceil(rows, kRmsChain)); }

template <typename TX, typename TR, int VEC, int K>
cudaError_t launch(const RmsParams& p, int wpr, long long* parts, cudaStream_t st) {
  constexpr int kRow = K * (2 * Slot<TR, VEC>::kBytes + Slot<TX, VEC>::kBytes);
  constexpr auto kern = rms_bwd<TX, TR, VEC, K>;
  const int teams = kRmsThreads / 32 / wpr;
  const size_t smem = std::max((size_t)rms_depth(kRow) * kRow * kRmsThreads, (size_t)K * VEC * 4 * wpr * 32);
  const int fit = std::min(8, ctas_per_sm<kern>(kRmsThreads, smem));
  long long grid = std::min<long long>(rms_ceil(p.rows, teams), 148LL * std::max(fit, 1));
  grid = std::max<long long>({1, grid, rms_ceil(p.rows, (long long)teams * kRmsChain)});
  *parts = grid;
  kern<<<(unsigned)grid, kRmsThreads, smem, st>>>(p, wpr);
  return cudaGetLastError();
}
template <typename TX, typename TR, int VEC>
cudaError_t run_vec(const RmsParams& p, long long* parts, float* stat, cudaStream_t st) {
  const RmsForm f = rms_form(p.C, VEC, kRmsMost / VEC);
  if constexpr (VEC >= 4) {
    if (f.k == 1) return launch<TX, TR, VEC, 1>(p, f.wpr, parts, st);
    if (f.k == 2) return launch<TX, TR, VEC, 2>(p, f.wpr, parts, st);
    if (f.k == 3) return launch<TX, TR, VEC, 3>(p, f.wpr, parts, st);
    if (f.k == 4) return launch<TX, TR, VEC, 4>(p, f.wpr, parts, st);
  }
  if constexpr (VEC == 4) {
    if (f.k == 5 || f.k == 6) return launch<TX, TR, VEC, 6>(p, f.wpr, parts, st);
    if (f.k > 6) return launch<TX, TR, VEC, 8>(p, f.wpr, parts, st);
  }
  if constexpr (VEC <= 2) {
    if (f.k > 0 && f.k * VEC <= 8) return launch<TX, TR, VEC, 8 / VEC>(p, f.wpr, parts, st);
    if (f.k > 0 && f.k * VEC <= 16) return launch<TX, TR, VEC, 16 / VEC>(p, f.wpr, parts, st);
    if (f.k > 0) return launch<TX, TR, VEC, 32 / VEC>(p, f.wpr, parts, st);
  }
  rms_bwd_long<TX, TR><<<(unsigned)std::min<long long>(p.rows, 148 * 4), 512, 0, st>>>(p, stat);
  if (p.part != nullptr) {
    *parts = rms_ceil(p.rows, kRmsChain);
    const dim3 grid((unsigned)rms_ceil(p.C, 32), (unsigned)std::min<long long>(*parts, 65535));
    rms_bwd_cols<TX, TR><<<grid, dim3(32, 8), 0, st>>>(p, stat);
  }
  return cudaGetLastError();
}
template <typename TX, typename TR>
cudaError_t run(const RmsParams& p, int vec, long long* parts, float* stat, cudaStream_t st) {
  constexpr int kFull = 16 / sizeof(TX);
  if (vec >= kFull) return run_vec<TX, TR, kFull>(p, parts, stat, st);
  if (vec >= 2) return run_vec<TX, TR, 2>(p, parts, stat, st);
  return run_vec<TX, TR, 1>(p, parts, stat, st);
}

size_t round256(size_t x) { return (x + 255) & ~size_t(255); }

}  // namespace
}  // namespace ssm

using namespace ssm;

extern "C" {

int ssm_rms_norm_bwd_workspace_size(int64_t rows, int64_t C, size_t* bytes) {
  if (bytes == nullptr) return fail(SSM_ERR_INVALID, "rms_norm: bytes is NULL");
  const ssm_view some = {bytes, SSM_F32, 0, 0, 0};
  if (int rc = rms_check(rows, C, some, ssm_view{}, nullptr, SSM_F32)) return rc;
  *bytes = round256((size_t)most_parts(rows) * C * 4) + round256((size_t)rows * 4) + 256;
  return SSM_OK;
}

int ssm_rms_norm_bwd(int64_t rows, int64_t C, ssm_view total, const void* weight, int32_t weight_dtype, float eps,
                     ssm_view dy, ssm_view dtotal, ssm_view dx, ssm_view dresidual, void* dweight, void* workspace,
                     size_t workspace_bytes, void* stream) {
  if (total.ptr == nullptr) return fail(SSM_ERR_INVALID, "rms_norm: the normed sum is required");
  if (int rc = rms_check(rows, C, dy, total, weight, weight_dtype)) return rc;
  if (dx.ptr == nullptr || dx.dtype != dy.dtype)
    return fail(dx.ptr == nullptr ? SSM_ERR_INVALID : SSM_ERR_DTYPE, "rms_norm: dx is required, in dy's dtype");
  if ((dtotal.ptr != nullptr && dtotal.dtype != total.dtype) || (dresidual.ptr != nullptr && dresidual.dtype != total.dtype))
    return fail(SSM_ERR_DTYPE, "rms_norm: the sum's and the residual's gradients must have the sum's dtype");
  size_t need = 0;
  ssm_rms_norm_bwd_workspace_size(rows, C, &need);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(SSM_ERR_WORKSPACE, "rms_norm: workspace of %lld bytes required, %lld given", (long long)need,
                (long long)workspace_bytes);
  RmsParams p = {};
  p.t = const_cast<void*>(total.ptr);
  p.ts = total.batch_stride;
  p.w = weight;
  p.wbf16 = weight_dtype == SSM_BF16;
  p.y = const_cast<void*>(dy.ptr);
  p.ys = dy.batch_stride;
  p.dt = dtotal.ptr;
  p.dts = dtotal.batch_stride;
  p.dx = const_cast<void*>(dx.ptr);
  p.dxs = dx.batch_stride;
  p.dr = const_cast<void*>(dresidual.ptr);
  p.drs = dresidual.batch_stride;
  p.rows = rows;
  p.C = (int)C;
  p.eps = eps;
  p.inv_c = 1.0f / (float)C;
  unsigned char* at = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~uintptr_t(255));
  p.part = dweight != nullptr ? reinterpret_cast<float*>(at) : nullptr;
  float* stat = reinterpret_cast<float*>(at + round256((size_t)most_parts(rows) * C * 4));
  const int xb = dy.dtype == SSM_BF16 ? 2 : 4, tb = total.dtype == SSM_BF16 ? 2 : 4;
  const int vec = rms_vec(C, xb, {{p.t, p.ts, tb}, {p.y, p.ys, xb}, {p.dt, p.dts, tb}, {p.dx, p.dxs, xb}, {p.dr, p.drs, tb}});
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  long long parts = 0;
  cudaError_t e = dy.dtype == SSM_F32      ? run<float, float>(p, vec, &parts, stat, st)
                  : total.dtype == SSM_F32 ? run<__nv_bfloat16, float>(p, vec, &parts, stat, st)
                                           : run<__nv_bfloat16, __nv_bfloat16>(p, vec, &parts, stat, st);
  if (e == cudaSuccess && dweight != nullptr) {
    const unsigned grid = (unsigned)rms_ceil(C, 32);
    if (weight_dtype == SSM_BF16)
      rms_dweight<<<grid, dim3(32, 8), 0, st>>>(p.part, parts, p.C, static_cast<__nv_bfloat16*>(dweight));
    else
      rms_dweight<<<grid, dim3(32, 8), 0, st>>>(p.part, parts, p.C, static_cast<float*>(dweight));
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) return fail(SSM_ERR_CUDA, "rms_norm backward launch failed (error %lld)", (long long)e);
  return SSM_OK;
}

}  // extern "C"
