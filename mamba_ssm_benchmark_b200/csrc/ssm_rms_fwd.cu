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

// the largest; a NaN only where all are
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Of a row whose largest |t w| is `big`: the scale, and what t w is multiplied by for e4m3.  y / scale is t w 448 / big, which
// the root does not enter: four roundings, 4 u.  With the product of the root and the scale's reciprocal, within 2 and 1 ulp, more
// values next to a border between two e4m3 went to the wrong one (8192 x 2560: 0.72 of a million, this way 0.57), and 8 bits of
// 16384 x 5120 without a residual took 81 us for 74.  A zero row, and one whose root overflowed, is 0 (0 x inf is NaN and fmaxf
// passes over it).
__device__ __forceinline__ float row_scale(float big, float rstd) { return fmaxf(big * rstd, kRmsTiny) / kE4m3Max; }
// false: t w is multiplied by rstd first, for the product of the two factors is out of range (a row about as small as kRmsTiny)
__device__ __forceinline__ bool row_factor(float big, float rstd, float& f) {
  const float top = big * rstd;
  if (top > kRmsTiny && top < __int_as_float(0x7f800000) && big > 1e-35f) {
    // 448 / big: a reciprocal of normal size, and one step of Newton's
    const float r = rcp(big * (1.0f / kE4m3Max));
    f = fmaf(fmaf(-r, big, kE4m3Max), r * (1.0f / kE4m3Max), r);
    return true;
  }
  const float inv = rcp(row_scale(big, rstd));
  f = rstd * inv;
  const bool fits = !(f > 1e38f);
  if (!fits) f = inv;
  return fits;
}

template <typename TX, typename TR, int VEC, int K, bool FP8, bool RAGGED>
__global__ void __launch_bounds__(kRmsThreads) rms_fwd(const __grid_constant__ RmsParams p, int wpr) {
  using SX = Slot<TX, VEC, RAGGED>;
  using SR = Slot<TR, VEC, RAGGED>;
  extern __shared__ __align__(16) unsigned char queue[];
  __shared__ float2 red[kRmsRed];
  Team team(wpr, red);
  const int warps = blockDim.x >> 5, teams = warps / wpr, lane = team.lane;
  constexpr int kStage = K * (SX::kWarp + SR::kWarp);     // a warp's bytes of a stage: K parts of x, K of the residual
  prefetch_weight(p);
  clear_queue(queue, warps * kRmsDepth * kStage);
  pdl_launch_dependents();
  pdl_wait();
  unsigned char* mine = queue + (threadIdx.x >> 5) * kRmsDepth * kStage;
  const long long step = (long long)gridDim.x * teams;
  long long row = (long long)blockIdx.x * teams + team.id;
  const bool adds = p.r != nullptr;
  auto c0 = [&](int k) { return (team.warp * 32 + k * team.size) * VEC; };
  auto fetch = [&](long long r, int stage) {
    unsigned char* at = mine + stage * kStage;
    if (r < p.rows) {
      const TX* x = static_cast<const TX*>(p.x) + r * p.xs;
      const TR* res = static_cast<const TR*>(p.r) + r * p.rs;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        SX::fetch(at + k * SX::kWarp, x, c0(k), p.C, lane);
        if (adds) SR::fetch(at + K * SX::kWarp + k * SR::kWarp, res, c0(k), p.C, lane);
      }
    }
    queue_commit();
  };
#pragma unroll
  for (int d = 0; d < kRmsDepth; ++d) fetch(row + d * step, d);
  float2 w[K][VEC / 2];
#pragma unroll
  for (int k = 0; k < K; ++k) load_weight<VEC>(p, c0(k) + lane * VEC, p.C - c0(k) - lane * VEC, w[k]);
  int stage = 0;
  for (; row < p.rows; row += step) {             // the same count for all warps of a team
    const TX* x = static_cast<const TX*>(p.x) + row * p.xs;
    const TR* res = static_cast<const TR*>(p.r) + row * p.rs;
    float2 v[K][VEC / 2], ss = make_float2(0.0f, 0.0f);
    queue_wait<kRmsDepth - 1>();
    __syncwarp();                                 // a lane reads what others fetched
    const unsigned char* at = mine + stage * kStage;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      SX::read(at + k * SX::kWarp, x, c0(k), lane, v[k]);
      if (adds) {
        float2 r[VEC / 2];
        uint32_t t[SR::kWords];
        SR::read(at + K * SX::kWarp + k * SR::kWarp, res, c0(k), lane, r);
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) v[k][i] = add2(v[k][i], r[i]);
        SR::pack(v[k], t);
        SR::write(static_cast<TR*>(p.t) + row * p.ts, c0(k), p.C, lane, t);
        SR::unpack(t, v[k]);                      // as it is kept
      }
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) ss = fma2(v[k][i], v[k][i], ss);
    }
    __syncwarp();
    fetch(row + kRmsDepth * step, stage);
    stage = stage + 1 == kRmsDepth ? 0 : stage + 1;
    float rstd = 1.0f;
    if (!FP8 || p.norm) {
      rstd = rsqrtf(team.sum(ss.x + ss.y) * p.inv_c + p.eps);      // within 2 ulp; a root and a quotient cost a row 40 instructions
      // in 8 bits rstd joins the scale: one product less
      const float2 f = bc2(FP8 ? 1.0f : rstd);
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) v[k][i] = FP8 ? mul2(v[k][i], w[k][i]) : mul2(mul2(v[k][i], f), w[k][i]);
    }
    if constexpr (FP8) {
      float big = 0.0f;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) big = max3(big, fabsf(v[k][i].x), fabsf(v[k][i].y));
      big = team.max(big);
      if (team.tid == 0) p.scale[row] = row_scale(big, rstd);
      float f;
      if (!row_factor(big, rstd, f)) {            // one factor after the other
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int i = 0; i < VEC / 2; ++i) v[k][i] = mul2(v[k][i], bc2(rstd));
      }
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = c0(k) + lane * VEC;
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) v[k][i] = mul2(v[k][i], bc2(f));
        if (c < p.C) write_e4m3<VEC>(static_cast<uint8_t*>(p.y) + row * p.ys + c, p.C - c, p.wide8, v[k]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        uint32_t y[SX::kWords];
        SX::pack(v[k], y);
        SX::write(static_cast<TX*>(p.y) + row * p.ys, c0(k), p.C, lane, y);
      }
    }
  }
  queue_wait<0>();
}

// Rows that no team holds (above 8192 channels): a CTA passes over the row for the sum
// of squares, for the largest value and for the result.
template <typename TX, typename TR, bool FP8>
__global__ void __launch_bounds__(kRmsThreads, 4) rms_fwd_long(const __grid_constant__ RmsParams p) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float2 red[kRmsRed];
  Team team(kRmsWarps, red);
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const TX* x = static_cast<const TX*>(p.x) + row * p.xs;
    TR* t = static_cast<TR*>(p.t) + row * p.ts;
    // a thread reads the sums that it wrote itself
    auto value = [&](int c) { return p.r != nullptr ? to_f32(t[c]) : to_f32(x[c]); };
    double ss = 0.0;
    by_fours(p.C, [&](int c, auto n) {
      float part = 0.0f;
      auto one = [&](int c, float v) {
        if (p.r != nullptr) {
          const TR sum = from_f32<TR>(v + to_f32(static_cast<const TR*>(p.r)[row * p.rs + c]));
          t[c] = sum;
          v = to_f32(sum);
        }
        part = fmaf(v, v, part);
      };
      // Loads ahead of the sums' stores (512 x 65536 bf16 95 us, one after another 104); in 8 bits the two more passes want their
      // registers (162 us, one after another 131).
      if constexpr (FP8) {
#pragma unroll
        for (int i = 0; i < n; ++i) one(c + i * kRmsThreads, to_f32(x[c + i * kRmsThreads]));
      } else {
        float v[n];
#pragma unroll
        for (int i = 0; i < n; ++i) v[i] = to_f32(x[c + i * kRmsThreads]);
#pragma unroll
        for (int i = 0; i < n; ++i) one(c + i * kRmsThreads, v[i]);
      }
      ss += (double)part;
    });
    const bool norm = !FP8 || p.norm;
    const float rstd = norm ? rsqrtf(team.sum((float)ss) * p.inv_c + p.eps) : 1.0f;
    // in 8 bits without rstd, which joins the scale
    auto result = [&](int c) {
      if (!norm) return value(c);
      return FP8 ? value(c) * weight_at(p, c) : value(c) * rstd * weight_at(p, c);
    };
    if constexpr (FP8) {
      float big = 0.0f, f;
      for (int c = threadIdx.x; c < p.C; c += 512) big = fmaxf(big, fabsf(result(c)));
      big = team.max(big);
      if (threadIdx.x == 0) p.scale[row] = row_scale(big, rstd);
      const float first = row_factor(big, rstd, f) ? 1.0f : rstd;
      for (int c = threadIdx.x; c < p.C; c += 512)
        static_cast<uint8_t*>(p.y)[row * p.ys + c] = __nv_cvt_float_to_fp8(result(c) * first * f, __NV_SATFINITE, __NV_E4M3);
    } else {
      for (int c = threadIdx.x; c < p.C; c += 512) static_cast<TX*>(p.y)[row * p.ys + c] = from_f32<TX>(result(c));
    }
  }
}

// ---- host -----------------------------------------------------------------------------------
template <typename TX, typename TR, int K, bool FP8, bool RAGGED>
cudaError_t launch(const RmsParams& p, RmsForm f, cudaStream_t st) {
  constexpr int VEC = 16 / sizeof(TX);
  using SX = Slot<TX, VEC, RAGGED>;
  using SR = Slot<TR, VEC, RAGGED>;
  constexpr auto kern = rms_fwd<TX, TR, VEC, K, FP8, RAGGED>;
  const int threads = f.threads();
  constexpr size_t warp = (size_t)kRmsDepth * K * (SX::kWarp + SR::kWarp);
  const size_t smem = warp * (threads / 32);
  const int fit = std::max(1, ctas_per_sm_threads<kern>(threads, smem, warp * kRmsWarps));
  const long long grid = std::min<long long>(rms_ceil(p.rows, f.teams()), 148LL * fit);
  return launch_pdl(kern, (unsigned)grid, threads, smem, st, p, f.wpr);
}
template <typename TX, typename TR, bool FP8, bool RAGGED>
cudaError_t run_form(const RmsParams& p, cudaStream_t st) {
  constexpr int VEC = 16 / sizeof(TX), kMany = kRmsMost / VEC;
  const RmsForm f = rms_form(p.C, VEC, {kMany, kMany / 2, 1});
  if (f.k == kMany) return launch<TX, TR, kMany, FP8, RAGGED>(p, f, st);
  if (VEC == 4 && f.k == 2) return launch<TX, TR, 2, FP8, RAGGED>(p, f, st);
  if (f.k == 1) return launch<TX, TR, 1, FP8, RAGGED>(p, f, st);
  return launch_pdl(rms_fwd_long<TX, TR, FP8>, (unsigned)std::min<long long>(p.rows, 148 * 4), kRmsThreads, 0, st, p);
}
template <typename TX, typename TR, bool FP8>
cudaError_t run(const RmsParams& p, bool aligned, cudaStream_t st) {
  return aligned ? run_form<TX, TR, FP8, false>(p, st) : run_form<TX, TR, FP8, true>(p, st);
}
template <bool FP8>
cudaError_t run_types(const RmsParams& p, int xd, int rd, bool aligned, cudaStream_t st) {
  if (xd == SSM_F32) return run<float, float, FP8>(p, aligned, st);
  if (rd == SSM_F32) return run<__nv_bfloat16, float, FP8>(p, aligned, st);
  return run<__nv_bfloat16, __nv_bfloat16, FP8>(p, aligned, st);
}

int fail(int code, const char* fmt, long long a = 0, long long b = 0) {
  char msg[256];
  snprintf(msg, sizeof(msg), fmt, a, b);
  return report_error(code, msg);
}

}  // namespace

// Whether rows are whole vectors that start at multiples of 16 bytes.
bool rms_aligned(long long C, int vec, std::initializer_list<RmsSide> sides) {
  bool fits = C % vec == 0;
  for (const RmsSide& s : sides)
    fits = fits && (s.ptr == nullptr || (reinterpret_cast<uintptr_t>(s.ptr) % 16 == 0 && s.stride * s.bytes % 16 == 0));
  return fits;
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
  const RmsSide out = {fp8 ? nullptr : p.y, p.ys, xb};
  const bool aligned = rms_aligned(C, 16 / xb, {{x.ptr, p.xs, xb}, {p.r, p.rs, rb}, {p.t, p.ts, rb}, out});
  p.wide8 = fp8 && ((reinterpret_cast<uintptr_t>(p.y) | (uintptr_t)p.ys) & 7) == 0;
  const int rd = residual.ptr != nullptr ? residual.dtype : x.dtype;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = fp8 ? run_types<true>(p, x.dtype, rd, aligned, st) : run_types<false>(p, x.dtype, rd, aligned, st);
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
