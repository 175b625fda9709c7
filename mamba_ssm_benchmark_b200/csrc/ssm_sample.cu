// ssm_sample.cu — the next token of every row of logits, from a given uniform number.
//
// Of w = exp((l - max) / temperature): the top_k largest are kept; of these, largest first, as many as it takes for their
// sum to reach top_p of all of theirs; of these what is at least min_p.  The token is the first, by index, where the running
// sum of the kept weights passes u times their sum.  Equal logits rank by index.
//
// A token must not depend on how sums are split, nor change when a sum's rounding does: weights are whole numbers in
// units of 2^-42, formed in double, and every sum is a 64-bit whole number, exact in any order (up to 2^20 tokens).  A weight
// is off by at most 2^-43 of the largest; what rounds to zero is never drawn.
//
// A cluster of up to eight CTAs shares a row, a slice of tokens each, kept in shared memory where it fits.
#include <cooperative_groups.h>

#include <algorithm>
#include <cstdio>

#include "ssm_b200.h"
#include "ssm_launch.cuh"
#include "ssm_vec.cuh"

namespace cg = cooperative_groups;

namespace ssm {
int report_error(int code, const char* msg);
}  // namespace ssm

namespace {

using u64 = unsigned long long;

struct SampleParams {
  const void* logits;
  long long stride;                   // of a row
  const float* u;
  const double *temperature, *top_p, *min_p;      // by row, or null: the values below
  const long long* top_k;
  double temperature0, top_p0, min_p0;
  long long top_k0;
  long long* token;
  int V, bf16;
  int slice;                          // tokens of a CTA
  int cached;                         // its logits are kept in shared memory
};

constexpr int kBits = 42;
constexpr u64 kOne = 1ull << kBits;
constexpr int kTable = 64;            // steps of the table of 2^x

struct SampleSmem {
  double exp2[kTable];
  u64 part[32], slot[2];
  float logits[1];                    // the slice
};

// A whole number that orders floats as they compare (-0 as 0); the index decides among equal ones, the lowest first.
__device__ __forceinline__ u64 rank_key(float l, int i) {
  const uint32_t b = __float_as_uint(l + 0.0f);
  return (u64)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (0xffffffffu - (uint32_t)i);
}
__device__ __forceinline__ float key_logit(u64 key) {
  const uint32_t b = (uint32_t)(key >> 32);
  return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}

struct Sampler {
  const SampleParams& p;
  SampleSmem& s;
  cg::cluster_group cluster;
  int row, ctas, lane, warp, first, last, turn;
  float top;                          // the largest logit
  double rate;                        // log2(e) / temperature

  __device__ Sampler(const SampleParams& p_, SampleSmem& s_) : p(p_), s(s_), cluster(cg::this_cluster()), turn(0) {
    ctas = (int)cluster.num_blocks();
    row = (int)blockIdx.x / ctas;
    lane = threadIdx.x & 31;
    warp = threadIdx.x >> 5;
  }
  __device__ float load(int i) const {
    return p.bf16 ? ssm::to_f32(static_cast<const __nv_bfloat16*>(p.logits)[row * p.stride + i])
                  : static_cast<const float*>(p.logits)[row * p.stride + i];
  }
  // A warp's tokens are neighbours, so that warps in order are tokens in order.
  __device__ void divide() {
    const int begin = min(p.V, (int)cluster.block_rank() * p.slice), end = min(p.V, begin + p.slice);
    const int warps = blockDim.x >> 5, per = ((end - begin + warps - 1) / warps + 31) & ~31;
    first = min(end, begin + warp * per);
    last = min(end, first + per);
    base = begin;
  }
  int base;
  __device__ float logit(int i) const { return p.cached ? s.logits[i - base] : load(i); }

  // 2^42 exp((l - top) / temperature).  2^y = 2^k 2^(j/64) 2^f, |f| <= 1/128: the Taylor polynomial of degree 5 is
  // within (ln 2 / 128)^6 / 720 = 4e-17 of 2^f.
  __device__ double weight(float l) const {
    if (l == top) return (double)kOne;
    const double y = ((double)l - (double)top) * rate;
    if (!(y > -(double)(kBits + 2))) return 0.0;           // below a quarter of a unit; also l = -inf
    constexpr double kShift = 6755399441055744.0 / kTable;   // 1.5 2^52 / 64: y is rounded to 64ths
    const double t = y + kShift;
    const int i = __double2loint(t);                       // 64 y, rounded
    const double f = (y - (t - kShift)) * 0.6931471805599453;
    double q = fma(f, 1.0 / 120, 1.0 / 24);
    q = fma(f, q, 1.0 / 6);
    q = fma(f, q, 0.5);
    q = fma(f, q, 1.0);
    q = fma(f, q, 1.0);
    const double scale = __hiloint2double((1023 + kBits + (i >> 6)) << 20, 0);
    return q * s.exp2[i & (kTable - 1)] * scale;
  }
  static __device__ u64 units(double w) { return (u64)__double_as_longlong(w + 4503599627370496.0) & ((1ull << 52) - 1); }

  // The sum (or maximum) over the cluster's threads, for all of them.
  template <bool MAX>
  __device__ u64 join(u64 v) {
    auto f = [](u64 a, u64 b) { return MAX ? (a > b ? a : b) : a + b; };
#pragma unroll
    for (int m = 16; m >= 1; m /= 2) v = f(v, __shfl_xor_sync(0xffffffffu, v, m));
    if (lane == 0) s.part[warp] = v;
    __syncthreads();
    v = lane < (int)(blockDim.x >> 5) ? s.part[lane] : 0;
#pragma unroll
    for (int m = 16; m >= 1; m /= 2) v = f(v, __shfl_xor_sync(0xffffffffu, v, m));
    if (ctas == 1) {
      __syncthreads();
      return v;
    }
    if (threadIdx.x == 0) s.slot[turn] = v;
    cluster.sync();
    v = 0;
    for (int r = 0; r < ctas; ++r) v = f(v, *cluster.map_shared_rank(&s.slot[turn], r));
    turn ^= 1;
    return v;
  }

  // How many tokens (or what weight) rank at least as high as both keys.
  template <bool MASS>
  __device__ u64 above(u64 cut, u64 key) {
    u64 n = 0;
    const u64 least = cut > key ? cut : key;
    for (int i = first + lane; i < last; i += 32) {
      const float l = logit(i);
      if (rank_key(l, i) >= least) n += MASS ? units(weight(l)) : 1;
    }
    return join<false>(n);
  }
  // The key of the token, by rank, at which the count (or weight) of those that rank at least as high as `cut`
  // reaches `target`; one that has all of them where it does not.
  template <bool MASS>
  __device__ u64 select(u64 cut, u64 target) {
    u64 lo = 0, hi = ~0ull;               // above(lo) >= target (or lo = 0), above(hi + 1) < target
    while (lo < hi) {
      const u64 mid = lo + (hi - lo) / 2 + 1;
      if (above<MASS>(cut, mid) >= target) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  }
};

__global__ void __launch_bounds__(1024) sample_tokens(const __grid_constant__ SampleParams p) {
  extern __shared__ __align__(16) unsigned char raw[];
  SampleSmem& s = *reinterpret_cast<SampleSmem*>(raw);
  Sampler a(p, s);
  a.divide();
  if (threadIdx.x < kTable) s.exp2[threadIdx.x] = exp2((double)threadIdx.x / kTable);
  const double temperature = p.temperature != nullptr ? p.temperature[a.row] : p.temperature0;
  const double top_p = p.top_p != nullptr ? p.top_p[a.row] : p.top_p0, min_p = p.min_p != nullptr ? p.min_p[a.row] : p.min_p0;
  const long long top_k = p.top_k != nullptr ? p.top_k[a.row] : p.top_k0;
  u64 best = 0;
  for (int i = a.first + a.lane; i < a.last; i += 32) {
    const float l = a.load(i);
    if (p.cached) s.logits[i - a.base] = l;
    const u64 key = l != l ? ~0ull : rank_key(l, i);      // a NaN ranks above all
    best = key > best ? key : best;
  }
  best = a.join<true>(best);
  a.top = key_logit(best);
  const bool none = best == ~0ull || a.top == -__int_as_float(0x7f800000) || temperature != temperature;
  const bool writes = threadIdx.x == 0 && a.cluster.block_rank() == 0;
  if (none || !(temperature > 0.0)) {                     // the same for the whole cluster
    if (writes) p.token[a.row] = none ? -1 : (long long)(0xffffffffu - (uint32_t)best);
    if (a.ctas > 1) a.cluster.sync();                     // peers read this CTA's slots until here
    return;
  }
  a.rate = 1.4426950408889634 / temperature;
  u64 cut = 0;
  if (top_k > 0 && top_k < p.V) cut = a.select<false>(cut, (u64)top_k);
  if (top_p < 1.0) {
    const double target = ceil(top_p * (double)a.above<true>(cut, 0));
    cut = max(cut, a.select<true>(cut, target > 1.0 ? (u64)target : 1));
  }
  const double least = fmin(fmax(min_p, 0.0), 1.0) * (double)kOne;
  auto kept = [&](int i) -> u64 {
    const float l = a.logit(i);
    if (rank_key(l, i) < cut) return 0;
    const double w = a.weight(l);
    return w >= least ? Sampler::units(w) : 0;
  };
  u64 mine = 0;
  for (int i = a.first + a.lane; i < a.last; i += 32) mine += kept(i);
  const u64 total = a.join<false>(mine);
  // what the warps and CTAs before have
  u64 sum = mine;
#pragma unroll
  for (int m = 16; m >= 1; m /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, m);
  if (a.lane == 0) s.part[a.warp] = sum;
  __syncthreads();
  u64 before = 0, cta = 0;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) {
    if (w < a.warp) before += s.part[w];
    cta += s.part[w];
  }
  if (a.ctas > 1) {
    if (threadIdx.x == 0) s.slot[a.turn] = cta;
    a.cluster.sync();
    for (int r = 0; r < (int)a.cluster.block_rank(); ++r) before += *a.cluster.map_shared_rank(&s.slot[a.turn], r);
  }
  const double at = (double)p.u[a.row] * (double)total;
  const u64 target = at > 0.0 ? min((u64)at, total - 1) : 0;
  if (before <= target && target < before + sum) {        // one warp of the cluster
    for (int i0 = a.first; i0 < a.last; i0 += 32) {
      u64 run = i0 + a.lane < a.last ? kept(i0 + a.lane) : 0;
#pragma unroll
      for (int m = 1; m < 32; m *= 2) {
        const u64 up = __shfl_up_sync(0xffffffffu, run, m);
        if (a.lane >= m) run += up;
      }
      const uint32_t passed = __ballot_sync(0xffffffffu, before + run > target);
      if (passed != 0) {
        if (a.lane == 0) p.token[a.row] = i0 + __ffs(passed) - 1;
        break;
      }
      before += __shfl_sync(0xffffffffu, run, 31);
    }
  }
  if (a.ctas > 1) a.cluster.sync();
}

// ---- host -----------------------------------------------------------------------------------
int fail(int code, const char* fmt, long long a = 0, long long b = 0) {
  char msg[256];
  snprintf(msg, sizeof(msg), fmt, a, b);
  return ssm::report_error(code, msg);
}
constexpr int kCached = 48 * 1024;    // logits that a CTA keeps

}  // namespace

extern "C" int ssm_sample_tokens(int64_t B, int64_t V, ssm_view logits, const float* uniforms, const double* temperature,
                                 double temperature0, const int64_t* top_k, int64_t top_k0, const double* top_p, double top_p0,
                                 const double* min_p, double min_p0, int64_t* tokens, void* stream) {
  if (B < 1 || V < 1) return fail(SSM_ERR_INVALID, "sample_tokens: rows and vocabulary must be positive");
  if (V > (1LL << 20) || B > (1LL << 27))
    return fail(SSM_ERR_INVALID, "sample_tokens: shape out of range (rows %lld, vocabulary %lld)", B, V);
  if (logits.ptr == nullptr || uniforms == nullptr || tokens == nullptr)
    return fail(SSM_ERR_INVALID, "sample_tokens: logits, uniforms and tokens are required");
  if (logits.dtype != SSM_F32 && logits.dtype != SSM_BF16)
    return fail(SSM_ERR_DTYPE, "sample_tokens: logits dtype %lld unsupported", logits.dtype);
  SampleParams p = {};
  p.logits = logits.ptr;
  p.stride = logits.batch_stride;
  p.bf16 = logits.dtype == SSM_BF16;
  p.u = uniforms;
  p.temperature = temperature;
  p.temperature0 = temperature0;
  p.top_k = reinterpret_cast<const long long*>(top_k);
  p.top_k0 = top_k0;
  p.top_p = top_p;
  p.top_p0 = top_p0;
  p.min_p = min_p;
  p.min_p0 = min_p0;
  p.token = reinterpret_cast<long long*>(tokens);
  p.V = (int)V;
  // CTAs to a row: what keeps the slices in shared memory, and more where few rows leave SMs idle
  int ctas = 1;
  while (ctas < 8 && V > (int64_t)ctas * kCached) ctas *= 2;
  while (ctas < 8 && V >= (int64_t)ctas * 8192 && B * ctas * 2 <= 148) ctas *= 2;
  p.slice = (int)((V + ctas - 1) / ctas);
  p.cached = p.slice <= kCached;
  const int threads = p.slice <= 128 ? 32 : p.slice <= 1024 ? 128 : p.slice <= 4096 ? 512 : 1024;
  ssm::ctas_per_sm<sample_tokens>(1024, sizeof(SampleSmem) + kCached * sizeof(float));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(B * ctas));
  cfg.blockDim = dim3((unsigned)std::max(threads, kTable));
  cfg.dynamicSmemBytes = sizeof(SampleSmem) + (p.cached ? p.slice * sizeof(float) : 0);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_tokens, p);
  return e == cudaSuccess ? SSM_OK : fail(SSM_ERR_CUDA, "sample_tokens launch failed (error %lld)", (long long)e);
}
