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

template <typename TX, typename TR, int VEC, int K, bool RAGGED>
__global__ void __launch_bounds__(kRmsThreads) rms_bwd(const __grid_constant__ RmsParams p, int wpr) {
  using ST = Slot<TR, VEC, RAGGED>;
  using SG = Slot<TX, VEC, RAGGED>;
  extern __shared__ __align__(16) unsigned char queue[];
  __shared__ float2 red[kRmsRed];
  Team team(wpr, red);
  const int warps = blockDim.x >> 5, teams = warps / wpr, lane = team.lane;
  // this warp's bytes of a stage: K parts of t, of dy, of dt
  constexpr int kG = K * ST::kWarp, kD = kG + K * SG::kWarp, kStage = kD + K * ST::kWarp;
  clear_queue(queue, warps * kRmsDepth * kStage);
  pdl_launch_dependents();
  pdl_wait();
  unsigned char* mine = queue + (threadIdx.x >> 5) * kRmsDepth * kStage;
  const long long step = (long long)gridDim.x * teams;
  long long row = (long long)blockIdx.x * teams + team.id;
  const bool adds = p.dt != nullptr;
  auto c0 = [&](int k) { return (team.warp * 32 + k * team.size) * VEC; };
  auto fetch = [&](long long r, int stage) {
    unsigned char* at = mine + stage * kStage;
    if (r < p.rows) {
      const TR* t = static_cast<const TR*>(p.t) + r * p.ts;
      const TX* g = static_cast<const TX*>(p.y) + r * p.ys;
      const TR* d = static_cast<const TR*>(p.dt) + r * p.dts;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        ST::fetch(at + k * ST::kWarp, t, c0(k), p.C, lane);
        SG::fetch(at + kG + k * SG::kWarp, g, c0(k), p.C, lane);
        if (adds) ST::fetch(at + kD + k * ST::kWarp, d, c0(k), p.C, lane);
      }
    }
    queue_commit();
  };
#pragma unroll
  for (int d = 0; d < kRmsDepth; ++d) fetch(row + d * step, d);
  float2 w[K][VEC / 2], dw[K][VEC / 2];
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) dw[k][i] = make_float2(0.0f, 0.0f);
    load_weight<VEC>(p, c0(k) + lane * VEC, p.C - c0(k) - lane * VEC, w[k]);
  }
  int stage = 0;
  for (; row < p.rows; row += step) {
    // The row is read from its slots twice: kept in registers between the sums and their use, it left 8 warps to an SM
    // (16384 x 5120 bf16: 150 us).
    const TR* t_row = static_cast<const TR*>(p.t) + row * p.ts;
    const TX* g_row = static_cast<const TX*>(p.y) + row * p.ys;
    const TR* d_row = static_cast<const TR*>(p.dt) + row * p.dts;
    float2 ss = make_float2(0.0f, 0.0f), gt = ss;
    queue_wait<kRmsDepth - 1>();
    __syncwarp();
    const unsigned char* at = mine + stage * kStage;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float2 t[VEC / 2], g[VEC / 2];
      ST::read(at + k * ST::kWarp, t_row, c0(k), lane, t);
      SG::read(at + kG + k * SG::kWarp, g_row, c0(k), lane, g);
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) {
        ss = fma2(t[i], t[i], ss);
        gt = fma2(mul2(g[i], w[k][i]), t[i], gt);
      }
    }
    const float2 s = team.sum(make_float2(ss.x + ss.y, gt.x + gt.y));
    const float rstd = rsqrtf(s.x * p.inv_c + p.eps);
    const float2 r2 = bc2(rstd), mean = bc2(-s.y * rstd * p.inv_c);      // minus that of g n
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float2 t[VEC / 2], g[VEC / 2], d[VEC / 2];
      ST::read(at + k * ST::kWarp, t_row, c0(k), lane, t);
      SG::read(at + kG + k * SG::kWarp, g_row, c0(k), lane, g);
      if (adds) {
        ST::read(at + kD + k * ST::kWarp, d_row, c0(k), lane, d);
      } else {
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) d[i] = make_float2(0.0f, 0.0f);
      }
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) {
        const float2 n = mul2(t[i], r2);
        dw[k][i] = fma2(g[i], n, dw[k][i]);
        d[i] = fma2(r2, fma2(n, mean, mul2(g[i], w[k][i])), d[i]);
      }
      uint32_t dx[SG::kWords];
      SG::pack(d, dx);
      SG::write(static_cast<TX*>(p.dx) + row * p.dxs, c0(k), p.C, lane, dx);
      if (p.dr != nullptr) {
        uint32_t dr[ST::kWords];
        ST::pack(d, dr);
        ST::write(static_cast<TR*>(p.dr) + row * p.drs, c0(k), p.C, lane, dr);
      }
    }
    __syncwarp();
    fetch(row + kRmsDepth * step, stage);
    stage = stage + 1 == kRmsDepth ? 0 : stage + 1;
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
          const float v = i & 1 ? dw[k][i / 2].y : dw[k][i / 2].x;
          s = q == 0 ? v : s + v;
        }
    }
  }
  if (team.id == teams - 1) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int c = c0(k) + lane * VEC + i;
        if (c < p.C) p.part[(size_t)blockIdx.x * p.C + c] = sum[(k * VEC + i) * team.size + team.tid];
      }
  }
}

// Rows that no team holds: a CTA per row for the sums and d; rstd goes to `stat`.
template <typename TX, typename TR>
__global__ void __launch_bounds__(kRmsThreads, 4) rms_bwd_long(const __grid_constant__ RmsParams p, float* stat) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float2 red[kRmsRed];
  Team team(kRmsWarps, red);
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const TR* t = static_cast<const TR*>(p.t) + row * p.ts;
    const TX* dy = static_cast<const TX*>(p.y) + row * p.ys;
    double ss = 0.0, gt = 0.0;
    by_fours(p.C, [&](int c, auto n) {
      float v[n], g[n];
      float2 part = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int i = 0; i < n; ++i) {
        v[i] = to_f32(t[c + i * kRmsThreads]);
        g[i] = to_f32(dy[c + i * kRmsThreads]) * weight_at(p, c + i * kRmsThreads);
      }
#pragma unroll
      for (int i = 0; i < n; ++i) part = make_float2(fmaf(v[i], v[i], part.x), fmaf(g[i], v[i], part.y));
      ss += (double)part.x;
      gt += (double)part.y;
    });
    const float2 s = team.sum(make_float2((float)ss, (float)gt));
    const float rstd = rsqrtf(s.x * p.inv_c + p.eps), mean = s.y * rstd * p.inv_c;
    if (threadIdx.x == 0) stat[row] = rstd;
    for (int c = threadIdx.x; c < p.C; c += 512) {
      const float d0 = p.dt != nullptr ? to_f32(static_cast<const TR*>(p.dt)[row * p.dts + c]) : 0.0f;
      const float d = fmaf(rstd, fmaf(-to_f32(t[c]) * rstd, mean, to_f32(dy[c]) * weight_at(p, c)), d0);
      static_cast<TX*>(p.dx)[row * p.dxs + c] = from_f32<TX>(d);
      if (p.dr != nullptr) static_cast<TR*>(p.dr)[row * p.drs + c] = from_f32<TR>(d);
    }
  }
}
// Their gradient of the weight: 32 channels and kRmsChain rows to a CTA, eight rows side by side.
template <typename TX, typename TR>
__global__ void __launch_bounds__(256) rms_bwd_cols(const __grid_constant__ RmsParams p, const float* stat) {
  pdl_launch_dependents();
  pdl_wait();
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
  pdl_launch_dependents();
  pdl_wait();
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
long long most_parts(long long rows) { return std::min(rows, std::max(kCtas, rms_ceil(rows, kRmsChain))); }

template <typename TX, typename TR, int K, bool RAGGED>
cudaError_t launch(const RmsParams& p, RmsForm f, long long* parts, cudaStream_t st) {
  constexpr int VEC = 16 / sizeof(TX);
  using ST = Slot<TR, VEC, RAGGED>;
  using SG = Slot<TX, VEC, RAGGED>;
  constexpr auto kern = rms_bwd<TX, TR, VEC, K, RAGGED>;
  const int threads = f.threads(), teams = f.teams();
  // the queue, which is larger than what the teams leave one another at the end
  constexpr size_t warp = (size_t)kRmsDepth * K * (2 * ST::kWarp + SG::kWarp);
  static_assert(warp >= (size_t)K * VEC * 4 * 32, "a team's gradients fit its part of the queue");
  const size_t smem = warp * (threads / 32);
  const int fit = std::min(8, std::max(1, ctas_per_sm_threads<kern>(threads, smem, warp * kRmsWarps)));
  // one wave, or as many as kRmsChain asks for
  const long long grid = std::max(std::min<long long>(rms_ceil(p.rows, teams), 148LL * fit),
                                  rms_ceil(p.rows, (long long)teams * kRmsChain));
  *parts = grid;
  return launch_pdl(kern, (unsigned)grid, threads, smem, st, p, f.wpr);
}
template <typename TX, typename TR, bool RAGGED>
cudaError_t run_form(const RmsParams& p, long long* parts, float* stat, cudaStream_t st) {
  constexpr int VEC = 16 / sizeof(TX), kMany = kRmsMost / VEC;
  const RmsForm f = rms_form(p.C, VEC, {kMany, kMany / 2, 1});
  if (f.k == kMany) return launch<TX, TR, kMany, RAGGED>(p, f, parts, st);
  if (VEC == 4 && f.k == 2) return launch<TX, TR, 2, RAGGED>(p, f, parts, st);
  if (f.k == 1) return launch<TX, TR, 1, RAGGED>(p, f, parts, st);
  cudaError_t e = launch_pdl(rms_bwd_long<TX, TR>, (unsigned)std::min<long long>(p.rows, 148 * 4), kRmsThreads, 0, st, p, stat);
  if (e == cudaSuccess && p.part != nullptr) {
    *parts = rms_ceil(p.rows, kRmsChain);
    const dim3 grid((unsigned)rms_ceil(p.C, 32), (unsigned)std::min<long long>(*parts, 65535));
    e = launch_pdl(rms_bwd_cols<TX, TR>, grid, dim3(32, 8), 0, st, p, stat);
  }
  return e;
}
template <typename TX, typename TR>
cudaError_t run(const RmsParams& p, bool aligned, long long* parts, float* stat, cudaStream_t st) {
  return aligned ? run_form<TX, TR, false>(p, parts, stat, st) : run_form<TX, TR, true>(p, parts, stat, st);
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
  const bool aligned = rms_aligned(
      C, 16 / xb, {{p.t, p.ts, tb}, {p.y, p.ys, xb}, {p.dt, p.dts, tb}, {p.dx, p.dxs, xb}, {p.dr, p.drs, tb}});
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  long long parts = 0;
  cudaError_t e = dy.dtype == SSM_F32      ? run<float, float>(p, aligned, &parts, stat, st)
                  : total.dtype == SSM_F32 ? run<__nv_bfloat16, float>(p, aligned, &parts, stat, st)
                                           : run<__nv_bfloat16, __nv_bfloat16>(p, aligned, &parts, stat, st);
  if (e == cudaSuccess && dweight != nullptr) {
    const unsigned grid = (unsigned)rms_ceil(C, 32);
    const dim3 block(32, 8);
    e = weight_dtype == SSM_BF16
            ? launch_pdl(rms_dweight<__nv_bfloat16>, grid, block, 0, st, p.part, parts, p.C, static_cast<__nv_bfloat16*>(dweight))
            : launch_pdl(rms_dweight<float>, grid, block, 0, st, p.part, parts, p.C, static_cast<float*>(dweight));
  }
  if (e != cudaSuccess) return fail(SSM_ERR_CUDA, "rms_norm backward launch failed (error %lld)", (long long)e);
  return SSM_OK;
}

}  // extern "C"
