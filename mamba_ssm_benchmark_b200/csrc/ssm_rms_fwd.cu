// ssm_rms_fwd.cu — forward of the root-mean-square norm with a residual, in the input's type or in 8 bits (ssm_rms.cuh).
//
// In 8 bits (e4m3) a row's values are y / scale with scale = max |y| / 448, one more butterfly over the row.
#include <cstdio>
#include <initializer_list>

#include "ssm_b200.h"
#include "ssm_rms.cuh"

namespace ssm {
int report_error(int code, const char* msg);

namespace {

template <typename TX, typename TR, int VEC, int K, bool FP8>
__global__ void __launch_bounds__(kRmsThreads) rms_fwd(const __grid_constant__ RmsParams p, int wpr) {
  constexpr int kRow = K * (Slot<TX, VEC>::kBytes + Slot<TR, VEC>::kBytes), kDepth = rms_depth(kRow);
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
      Slot<TX, VEC>::fetch(at + (size_t)k * Slot<TX, VEC>::kBytes * nt, static_cast<const TX*>(p.x) + (ok ? r * p.xs + c : 0), ok);
      if (p.r != nullptr)
        Slot<TR, VEC>::fetch(at + (size_t)(K * Slot<TX, VEC>::kBytes + k * Slot<TR, VEC>::kBytes) * nt,
                             static_cast<const TR*>(p.r) + (ok ? r * p.rs + c : 0), ok);
    }
    queue_commit();
  };
#pragma unroll
  for (int d = 0; d < kDepth; ++d) fetch(row + d * step, d);
  float w[K][VEC];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (team.tid + k * team.size) * VEC;
    if (c < p.C) load_weight<VEC>(p, c, w[k]);
  }
  int stage = 0;
  for (; row < p.rows; row += step) {             // the same count for all warps of a team
    float v[K][VEC];
    float ss = 0.0f;
    queue_wait<kDepth - 1>();
    const unsigned char* at = queue + (size_t)stage * kRow * nt;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (team.tid + k * team.size) * VEC;
      Slot<TX, VEC>::read(at + (size_t)k * Slot<TX, VEC>::kBytes * nt, v[k]);
      if (p.r != nullptr) {
        float r[VEC];
        Slot<TR, VEC>::read(at + (size_t)(K * Slot<TX, VEC>::kBytes + k * Slot<TR, VEC>::kBytes) * nt, r);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[k][i] = to_f32(from_f32<TR>(v[k][i] + r[i]));   // t as it is kept
        if (c < p.C) write_piece<TR, VEC>(static_cast<TR*>(p.t) + row * p.ts + c, v[k]);
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) ss = fmaf(v[k][i], v[k][i], ss);
    }
    fetch(row + kDepth * step, stage);
    stage = stage + 1 == kDepth ? 0 : stage + 1;
    if (!FP8 || p.norm) {
      const float rstd = 1.0f / sqrtf(team.sum(ss, 0.0f).x * p.inv_c + p.eps);
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[k][i] = v[k][i] * rstd * w[k][i];
    }
    if constexpr (FP8) {
      float big = 0.0f;
#pragma unroll
      for (int k = 0; k < K; ++k)
        if ((team.tid + k * team.size) * VEC < p.C) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) big = fmaxf(big, fabsf(v[k][i]));
        }
      const float scale = fmaxf(team.max(big), kRmsTiny) / kE4m3Max, inv = 1.0f / scale;
      if (team.tid == 0) p.scale[row] = scale;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (team.tid + k * team.size) * VEC;
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[k][i] *= inv;
        if (c < p.C) write_e4m3<VEC>(static_cast<uint8_t*>(p.y) + row * p.ys + c, v[k]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (team.tid + k * team.size) * VEC;
        if (c < p.C) write_piece<TX, VEC>(static_cast<TX*>(p.y) + row * p.ys + c, v[k]);
      }
    }
  }
  queue_wait<0>();
}

// Rows that no team holds (above 8192 channels): a CTA passes over the row for the sum
// of squares, for the largest value and for the result.
template <typename TX, typename TR, bool FP8>
__global__ void __launch_bounds__(512) rms_fwd_long(const __grid_constant__ RmsParams p) {
  __shared__ float2 red[2 * 16];
  Team team(16, red);
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const TX* x = static_cast<const TX*>(p.x) + row * p.xs;
    TR* t = static_cast<TR*>(p.t) + row * p.ts;
    // a thread reads the sums that it wrote itself
    auto value = [&](int c) { return p.r != nullptr ? to_f32(t[c]) : to_f32(x[c]); };
    float ss = 0.0f;
    for (int c = threadIdx.x; c < p.C; c += 512) {
      if (p.r != nullptr) t[c] = from_f32<TR>(to_f32(x[c]) + to_f32(static_cast<const TR*>(p.r)[row * p.rs + c]));
      const float v = value(c);
      ss = fmaf(v, v, ss);
    }
    const bool norm = !FP8 || p.norm;
    const float rstd = norm ? 1.0f / sqrtf(team.sum(ss, 0.0f).x * p.inv_c + p.eps) : 1.0f;
    auto result = [&](int c) {
      if (!norm) return value(c);
      float w[1];
      load_weight<1>(p, c, w);
      return value(c) * rstd * w[0];
    };
    if constexpr (FP8) {
      float big = 0.0f;
      for (int c = threadIdx.x; c < p.C; c += 512) big = fmaxf(big, fabsf(result(c)));
      const float scale = fmaxf(team.max(big), kRmsTiny) / kE4m3Max, inv = 1.0f / scale;
      if (threadIdx.x == 0) p.scale[row] = scale;
      for (int c = threadIdx.x; c < p.C; c += 512)
        static_cast<uint8_t*>(p.y)[row * p.ys + c] = __nv_cvt_float_to_fp8(result(c) * inv, __NV_SATFINITE, __NV_E4M3);
    } else {
      for (int c = threadIdx.x; c < p.C; c += 512) static_cast<TX*>(p.y)[row * p.ys + c] = from_f32<TX>(result(c));
    }
  }
}

// ---- host -----------------------------------------------------------------------------------
template <typename TX, typename TR, int VEC, int K, bool FP8>
cudaError_t launch(const RmsParams& p, int wpr, cudaStream_t st) {
  constexpr int kRow = K * (Slot<TX, VEC>::kBytes + Slot<TR, VEC>::kBytes);
  constexpr auto kern = rms_fwd<TX, TR, VEC, K, FP8>;
  const int teams = kRmsThreads / 32 / wpr;
  const size_t smem = (size_t)rms_depth(kRow) * kRow * kRmsThreads;
  const int fit = ctas_per_sm<kern>(kRmsThreads, smem);
  const long long grid = std::max<long long>(1, std::min<long long>(rms_ceil(p.rows, teams), 148LL * std::max(fit, 1)));
  kern<<<(unsigned)grid, kRmsThreads, smem, st>>>(p, wpr);
  return cudaGetLastError();
}
template <typename TX, typename TR, int VEC, bool FP8>
cudaError_t run_vec(const RmsParams& p, cudaStream_t st) {
  const RmsForm f = rms_form(p.C, VEC, kRmsMost / VEC);
  if constexpr (VEC >= 4) {
    if (f.k == 1) return launch<TX, TR, VEC, 1, FP8>(p, f.wpr, st);
    if (f.k == 2) return launch<TX, TR, VEC, 2, FP8>(p, f.wpr, st);
    if (f.k == 3) return launch<TX, TR, VEC, 3, FP8>(p, f.wpr, st);
    if (f.k == 4) return launch<TX, TR, VEC, 4, FP8>(p, f.wpr, st);
  }
  if constexpr (VEC == 4) {
    if (f.k == 5 || f.k == 6) return launch<TX, TR, VEC, 6, FP8>(p, f.wpr, st);
    if (f.k > 6) return launch<TX, TR, VEC, 8, FP8>(p, f.wpr, st);
  }
  if constexpr (VEC <= 2) {
    if (f.k > 0 && f.k * VEC <= 8) return launch<TX, TR, VEC, 8 / VEC, FP8>(p, f.wpr, st);
    if (f.k > 0 && f.k * VEC <= 16) return launch<TX, TR, VEC, 16 / VEC, FP8>(p, f.wpr, st);
    if (f.k > 0) return launch<TX, TR, VEC, 32 / VEC, FP8>(p, f.wpr, st);
  }
  rms_fwd_long<TX, TR, FP8><<<(unsigned)std::min<long long>(p.rows, 148 * 4), 512, 0, st>>>(p);
  return cudaGetLastError();
}
template <typename TX, typename TR, bool FP8>
cudaError_t run(const RmsParams& p, int vec, cudaStream_t st) {
  constexpr int kFull = 16 / sizeof(TX);
  if (vec >= kFull) return run_vec<TX, TR, kFull, FP8>(p, st);
  if (vec >= 2) return run_vec<TX, TR, 2, FP8>(p, st);
  return run_vec<TX, TR, 1, FP8>(p, st);
}
template <bool FP8>
cudaError_t run_types(const RmsParams& p, int xd, int rd, int vec, cudaStream_t st) {
  if (xd == SSM_F32) return run<float, float, FP8>(p, vec, st);
  if (rd == SSM_F32) return run<__nv_bfloat16, float, FP8>(p, vec, st);
  return run<__nv_bfloat16, __nv_bfloat16, FP8>(p, vec, st);
}

int fail(int code, const char* fmt, long long a = 0, long long b = 0) {
  char msg[256];
  snprintf(msg, sizeof(msg), fmt, a, b);
  return report_error(code, msg);
}

}  // namespace

// The widest vector (a power of two, at most 16 bytes of x) that divides the channels and at which every row starts
// aligned to a vector, or to 16 bytes.
int rms_vec(long long C, int xbytes, std::initializer_list<RmsSide> sides) {
  int vec = 16 / xbytes;
  while (C % vec != 0) vec /= 2;
  for (const RmsSide& s : sides) {
    if (s.ptr == nullptr) continue;
    while (vec > 1 && (reinterpret_cast<uintptr_t>(s.ptr) % std::min(16, vec * s.bytes) != 0 ||
                       s.stride * s.bytes % std::min(16, vec * s.bytes) != 0))
      vec /= 2;
  }
  return vec;
}

int rms_check(int64_t rows, int64_t C, const ssm_view& x, const ssm_view& residual, const void* weight, int32_t wdtype) {
  if (rows < 1 || C < 1) return fail(SSM_ERR_INVALID, "rms_norm: rows and channels must be positive");
  if (C > (1LL << 24) || rows > (1LL << 40) / C)
    return fail(SSM_ERR_INVALID, "rms_norm: shape out of range (rows %lld, channels %lld)", rows, C);
  if (x.ptr == nullptr) return fail(SSM_ERR_INVALID, "rms_norm: x is required");
  if (x.dtype != SSM_F32 && x.dtype != SSM_BF16) return fail(SSM_ERR_DTYPE, "rms_norm: x dtype %lld unsupported", x.dtype);
  if (residual.ptr != nullptr && residual.dtype != SSM_F32 && residual.dtype != x.dtype)
    return fail(SSM_ERR_DTYPE, "rms_norm: the residual must be float32 or have x's dtype");
  if (weight != nullptr && wdtype != SSM_F32 && wdtype != SSM_BF16)
    return fail(SSM_ERR_DTYPE, "rms_norm: weight dtype %lld unsupported", wdtype);
  return SSM_OK;
}

}  // namespace ssm

using namespace ssm;

static int forward(int64_t rows, int64_t C, ssm_view x, ssm_view residual, const void* weight, int32_t wdtype, float eps,
                   ssm_view y, uint8_t* y8, int64_t y8_stride, float* scale, int32_t norm, ssm_view total, void* stream) {
  if (int rc = rms_check(rows, C, x, residual, weight, wdtype)) return rc;
  const bool fp8 = y8 != nullptr;
  if (!fp8 && (y.ptr == nullptr || y.dtype != x.dtype))
    return fail(y.ptr == nullptr ? SSM_ERR_INVALID : SSM_ERR_DTYPE, "rms_norm: y is required, in x's dtype");
  if (residual.ptr != nullptr && (total.ptr == nullptr || total.dtype != residual.dtype))
    return fail(total.ptr == nullptr ? SSM_ERR_INVALID : SSM_ERR_DTYPE, "rms_norm: the sum is required, in the residual's dtype");
  RmsParams p = {};
  p.x = x.ptr;
  p.xs = x.batch_stride;
  p.r = residual.ptr;
  p.rs = residual.batch_stride;
  p.w = weight;
  p.wbf16 = wdtype == SSM_BF16;
  p.y = fp8 ? static_cast<void*>(y8) : const_cast<void*>(y.ptr);
  p.ys = fp8 ? y8_stride : y.batch_stride;
  p.t = residual.ptr != nullptr ? const_cast<void*>(total.ptr) : nullptr;
  p.ts = total.batch_stride;
  p.scale = scale;
  p.rows = rows;
  p.C = (int)C;
  p.eps = eps;
  p.inv_c = 1.0f / (float)C;
  p.norm = norm;
  const int xb = x.dtype == SSM_BF16 ? 2 : 4, rb = residual.dtype == SSM_BF16 ? 2 : 4;
  const int vec = rms_vec(C, xb, {{x.ptr, p.xs, xb}, {p.r, p.rs, rb}, {p.t, p.ts, rb}, {p.y, p.ys, fp8 ? 1 : xb}});
  const int rd = residual.ptr != nullptr ? residual.dtype : x.dtype;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = fp8 ? run_types<true>(p, x.dtype, rd, vec, st) : run_types<false>(p, x.dtype, rd, vec, st);
  if (e != cudaSuccess) return fail(SSM_ERR_CUDA, "rms_norm forward launch failed (error %lld)", (long long)e);
  return SSM_OK;
}

extern "C" {

int ssm_rms_norm_fwd(int64_t rows, int64_t C, ssm_view x, ssm_view residual, const void* weight, int32_t weight_dtype,
                     float eps, ssm_view y, ssm_view total, void* stream) {
  return forward(rows, C, x, residual, weight, weight_dtype, eps, y, nullptr, 0, nullptr, 1, total, stream);
}

int ssm_rms_norm_fp8(int64_t rows, int64_t C, ssm_view x, ssm_view residual, const void* weight, int32_t weight_dtype,
                     float eps, int32_t norm, void* y8, int64_t y8_stride, float* scale, ssm_view total, void* stream) {
  if (y8 == nullptr || scale == nullptr) return fail(SSM_ERR_INVALID, "rms_norm: y8 and scale are required");
  return forward(rows, C, x, residual, weight, weight_dtype, eps, ssm_view{}, static_cast<uint8_t*>(y8), y8_stride, scale,
                 norm, total, stream);
}

}  // extern "C"
