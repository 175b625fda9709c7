// ssm_linear8.cu — products of 8-bit rows (e4m3, a float32 scale for every row) with everything behind them.
//
//   y[m, n] = act(x_scale[m] w_scale[n] sum_k x8[m, k] w8[n, k] + bias[n]) + residual[m, n]
//
// The weight's 128 rows are the M of tcgen05.mma (lanes of tensor memory), 16 to 256 tokens its N (columns): one form
// serves a single token and a prompt, the weight's scale and bias are one value a thread, and 32 lanes store 32
// neighbouring channels.  TMA brings 128-byte K blocks of both (128-byte swizzle; what lies past an edge is zero); a warp
// copies, a warp multiplies, four warps read the accumulators of one tile while the next is multiplied.  Few tiles:
// the CTAs of a cluster take a part of K each and add their sums, in order, through distributed shared memory.
#include <algorithm>
#include <cstdio>

#include "ssm_b200.h"
#include "ssm_delta_tc.cuh"
#include "ssm_launch.cuh"

namespace ssm {
int report_error(int code, const char* msg);
int* device_error_word();
bool encode_rows8(CUtensorMap* map, const void* ptr, int64_t rows, int64_t cols, int64_t stride, int box_rows);
}  // namespace ssm

namespace {

using namespace ssm;

struct alignas(64) LinearParams {
  CUtensorMap tw, tx;
  const float *w_scale, *x_scale, *bias;      // bias may be null
  const void* res;                            // null, or like y
  void* y;
  long long rs, ys;                           // row strides
  int tokens, channels, blocks;               // blocks of K
  int tiles_n, tiles;                         // tiles over the channels, and in all
  int silu;
  int* err;
};

constexpr int kRowsW = 128, kBlockK = 128, kLinThreads = 192;

template <int TN>
struct LinearForm {
  static constexpr int kStage = (kRowsW + TN) * kBlockK;
  // TN <= 64: two CTAs share an SM; above, one with as many stages as fit
  static constexpr int kStages = TN <= 32 ? 5 : TN == 64 ? 4 : TN == 128 ? 6 : 4;
  static constexpr uint32_t kCols = 2 * TN;
  static constexpr size_t kSmem = (size_t)kStages * kStage + 1024 + 256;
};
template <int TN>
struct LinearBars {
  uint64_t full[LinearForm<TN>::kStages], empty[LinearForm<TN>::kStages], acc_full[2], acc_empty[2];
  uint32_t tmem;
};

__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
                   smem_u32(dst)),
               "l"(map), "r"(c0), "r"(c1), "r"(smem_u32(bar))
               : "memory");
}
// D (128 x N, fp32) (+)= A (128 x 32 e4m3) x B (N x 32 e4m3)^T, both in shared memory; see tc_mma.
__device__ __forceinline__ void tc_mma_e4m3(uint32_t d, uint32_t a, uint32_t b, uint32_t high, uint32_t idesc, bool accumulate,
                                            uint32_t issue) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(high), "r"(idesc), "r"((uint32_t)accumulate), "r"(issue)
      : "memory");
}
__device__ __forceinline__ void cluster_arrive_wait() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ float peer_load(uint32_t addr, uint32_t rank) {
  uint32_t at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

// y's value from an accumulator, the token's scale and the residual.
__device__ __forceinline__ float finish(const LinearParams& p, float acc, float w_scale, float x_scale, float bias, float res) {
  float v = fmaf(acc, w_scale * x_scale, bias);
  if (p.silu) v = v / (1.0f + __expf(-v));
  return v + res;
}

// SPLIT: a cluster takes one tile, its CTAs a part of K each.
template <int TN, typename TY, bool SPLIT>
__global__ void __launch_bounds__(kLinThreads) linear_e4m3(const __grid_constant__ LinearParams p, int parts) {
  using Form = LinearForm<TN>;
  constexpr int kStages = Form::kStages;
  extern __shared__ unsigned char raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  auto& bar = *reinterpret_cast<LinearBars<TN>*>(smem + (size_t)kStages * Form::kStage);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&bar.full[i], 1);
      mbar_init(&bar.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar.acc_full[i], 1);
      mbar_init(&bar.acc_empty[i], 4);
    }
    fence_mbar_init();
  }
  if (warp == 5) tc_alloc(&bar.tmem, Form::kCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = __shfl_sync(0xffffffffu, bar.tmem, 0);
  const int rank = SPLIT ? (int)cluster_rank() : 0;
  const int first = SPLIT ? (int)blockIdx.x / parts : (int)blockIdx.x, step = SPLIT ? p.tiles : (int)gridDim.x;
  const int k0 = SPLIT ? (int)((long long)p.blocks * rank / parts) : 0;
  const int k1 = SPLIT ? (int)((long long)p.blocks * (rank + 1) / parts) : p.blocks;
  Wait wait{p.err};
  if (warp == 4) {                                       // copies
    if (lane == 0) {
      int st = 0, par = 1;
      for (int t = first; t < p.tiles && !wait.dead; t += step) {
        const int n0 = t % p.tiles_n * kRowsW, m0 = t / p.tiles_n * TN;
        for (int k = k0; k < k1; ++k) {
          wait(&bar.empty[st], par);
          if (wait.dead) break;
          unsigned char* at = smem + (size_t)st * Form::kStage;
          mbar_arrive_expect_tx(&bar.full[st], Form::kStage);
          tma_load_2d(at, &p.tw, &bar.full[st], k * kBlockK, n0);
          tma_load_2d(at + kRowsW * kBlockK, &p.tx, &bar.full[st], k * kBlockK, m0);
          if (++st == kStages) st = 0, par ^= 1;
        }
      }
    }
    __syncwarp();
  } else if (warp == 5) {                                // products
    const uint32_t issue = lane == 0;
    // fp32 accumulators, both operands e4m3 and read along their rows, M = 128
    const uint32_t idesc = 1u << 4 | (uint32_t)(TN / 8) << 17 | (kRowsW / 16u) << 24;
    int st = 0, par = 0, buf = 0, bpar = 1;
    for (int t = first; t < p.tiles && !wait.dead; t += step) {
      wait(&bar.acc_empty[buf], bpar);
      tc_fence_after();
      const uint32_t d = tm + buf * TN;
      bool more = false;
      for (int k = k0; k < k1; ++k) {
        wait(&bar.full[st], par);
        wait.dead = __any_sync(0xffffffffu, wait.dead);
        if (wait.dead) break;
        tc_fence_after();
        const uint32_t a = tc_desc(smem_u32(smem + (size_t)st * Form::kStage), 16), b = a + kRowsW * kBlockK / 16;
#pragma unroll
        for (int i = 0; i < kBlockK / 32; ++i) {
          tc_mma_e4m3(d, a + 2 * i, b + 2 * i, kTcDescHigh, idesc, more, issue);
          more = true;
        }
        if (issue) tc_commit(&bar.empty[st]);
        if (++st == kStages) st = 0, par ^= 1;
      }
      if (issue && !wait.dead) tc_commit(&bar.acc_full[buf]);
      if (++buf == 2) buf = 0, bpar ^= 1;
    }
    __syncwarp();
  } else {                                               // results
    const uint32_t my = tm + ((uint32_t)(32 * warp) << 16);
    const int row = 32 * warp + lane;
    int buf = 0, bpar = 0;
    for (int t = first; t < p.tiles && !wait.dead; t += step) {
      const int n = t % p.tiles_n * kRowsW + row, m0 = t / p.tiles_n * TN;
      const bool live = n < p.channels;
      const float ws = live ? p.w_scale[n] : 0.0f, bias = live && p.bias != nullptr ? p.bias[n] : 0.0f;
      wait(&bar.acc_full[buf], bpar);
      wait.dead = __any_sync(0xffffffffu, wait.dead);
      if (!SPLIT && wait.dead) break;
      tc_fence_after();
      if constexpr (SPLIT) {                             // [column][row], over the stages: all products are done
        float* part = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int c = 0; c < TN; c += 16) {
          float v[16];
          tc_load_f32(my + buf * TN + c, v);
#pragma unroll
          for (int i = 0; i < 16; ++i) part[(c + i) * kRowsW + row] = wait.dead ? quiet_nan() : v[i];
        }
      } else {
        // 16 tokens at a time, the next ones' residuals on their way
        const TY* rp = static_cast<const TY*>(p.res) + (long long)m0 * p.rs + n;
        TY* yp = static_cast<TY*>(p.y) + (long long)m0 * p.ys + n;
        const bool adds = p.res != nullptr && live;
        TY next[16];
        auto fetch = [&](int c) {
#pragma unroll
          for (int i = 0; i < 16; ++i) next[i] = adds && m0 + c + i < p.tokens ? rp[(long long)(c + i) * p.rs] : from_f32<TY>(0.0f);
        };
        fetch(0);
#pragma unroll 2
        for (int c = 0; c < TN; c += 16) {
          const float xs = m0 + c + (lane & 15) < p.tokens ? p.x_scale[m0 + c + (lane & 15)] : 0.0f;
          float v[16];
          tc_load_f32(my + buf * TN + c, v);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            v[i] = finish(p, v[i], ws, __shfl_sync(0xffffffffu, xs, i), bias, to_f32(next[i]));
          if (c + 16 < TN) fetch(c + 16);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (live && m0 + c + i < p.tokens) yp[(long long)(c + i) * p.ys] = from_f32<TY>(v[i]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) tc_arrive(&bar.acc_empty[buf]);
      if (++buf == 2) buf = 0, bpar ^= 1;
    }
  }
  if constexpr (SPLIT) {
    __syncwarp();
    cluster_arrive_wait();
    if (warp < 4) {
      const int n = first % p.tiles_n * kRowsW + 32 * warp + lane, m0 = first / p.tiles_n * TN;
      if (n < p.channels) {
        const float ws = p.w_scale[n], bias = p.bias != nullptr ? p.bias[n] : 0.0f;
        // this CTA's columns, kJoin at a time so that as many loads are on their way
        constexpr int kJoin = TN >= 64 ? 8 : TN / 8;
        const int own = TN / parts;
        for (int c0 = rank * own; c0 < (rank + 1) * own && m0 + c0 < p.tokens; c0 += kJoin) {
          float v[kJoin], res[kJoin], xs[kJoin];
#pragma unroll
          for (int i = 0; i < kJoin; ++i) {
            const long long m = m0 + c0 + i;
            const bool in = m < p.tokens;
            xs[i] = in ? p.x_scale[m] : 0.0f;
            res[i] = in && p.res != nullptr ? to_f32(static_cast<const TY*>(p.res)[m * p.rs + n]) : 0.0f;
            v[i] = 0.0f;
          }
          for (int q = 0; q < parts; ++q) {
#pragma unroll
            for (int i = 0; i < kJoin; ++i) v[i] += peer_load(smem_u32(smem) + ((c0 + i) * kRowsW + 32 * warp + lane) * 4, q);
          }
#pragma unroll
          for (int i = 0; i < kJoin; ++i)
            if (m0 + c0 + i < p.tokens)
              static_cast<TY*>(p.y)[(m0 + c0 + i) * p.ys + n] = from_f32<TY>(finish(p, v[i], ws, xs[i], bias, res[i]));
        }
      }
    }
    __syncwarp();
    cluster_arrive_wait();                               // peers read this CTA's sums until here
  }
  wait.drain();
  __syncthreads();
  if (warp == 5) tc_free(tm, Form::kCols);
}

// ---- host -----------------------------------------------------------------------------------
int fail(int code, const char* fmt, long long a = 0, long long b = 0) {
  char msg[256];
  snprintf(msg, sizeof(msg), fmt, a, b);
  return report_error(code, msg);
}
int ceil_div(int a, int b) { return (a + b - 1) / b; }

template <int TN, typename TY, bool SPLIT>
cudaError_t launch(const LinearParams& p, int ctas, int parts, cudaStream_t st) {
  constexpr auto kern = linear_e4m3<TN, TY, SPLIT>;
  ctas_per_sm<kern>(kLinThreads, LinearForm<TN>::kSmem);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kLinThreads);
  cfg.dynamicSmemBytes = LinearForm<TN>::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = SPLIT ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, p, parts);
}

template <int TN, typename TY>
cudaError_t run(LinearParams& p, cudaStream_t st) {
  p.tiles_n = ceil_div(p.channels, kRowsW);
  p.tiles = p.tiles_n * ceil_div(p.tokens, TN);
  const int room = 148 * (TN <= 64 ? 2 : 1);
  int parts = 1;                                         // divides TN by kJoin or more
  while (parts < 8 && p.tiles * parts * 2 <= room && parts * 2 <= p.blocks) parts *= 2;
  if (parts > 1) return launch<TN, TY, true>(p, p.tiles * parts, parts, st);
  return launch<TN, TY, false>(p, std::min(p.tiles, room), 1, st);
}
template <typename TY>
cudaError_t run_tokens(LinearParams& p, int tn, cudaStream_t st) {
  if (tn == 16) return run<16, TY>(p, st);
  if (tn == 32) return run<32, TY>(p, st);
  if (tn == 64) return run<64, TY>(p, st);
  if (tn == 128) return run<128, TY>(p, st);
  return run<256, TY>(p, st);
}
int tile_tokens(int64_t tokens) {
  int tn = 16;
  while (tn < 256 && tn < tokens) tn *= 2;
  return tn;
}

}  // namespace

extern "C" {

int ssm_linear_fp8(int64_t tokens, int64_t channels, int64_t K, const void* x8, int64_t x_stride, const float* x_scale,
                   const void* w8, int64_t w_stride, const float* w_scale, const float* bias, int32_t silu,
                   ssm_view residual, ssm_view y, void* stream) {
  if (tokens < 1 || channels < 1 || K < 1)
    return fail(SSM_ERR_INVALID, "linear_fp8: tokens, channels and K must be positive");
  if (tokens > (1 << 28) || channels > (1 << 24) || K > (1 << 24) ||
      (channels + 127) / 128 * ((tokens + 15) / 16) > 0x7fffffffLL / 8)
    return fail(SSM_ERR_INVALID, "linear_fp8: shape out of range (tokens %lld, channels %lld)", tokens, channels);
  if (x8 == nullptr || x_scale == nullptr || w8 == nullptr || w_scale == nullptr || y.ptr == nullptr)
    return fail(SSM_ERR_INVALID, "linear_fp8: x8, w8, their scales and y are required");
  if (((reinterpret_cast<uintptr_t>(x8) | reinterpret_cast<uintptr_t>(w8) | (uintptr_t)x_stride | (uintptr_t)w_stride) & 15) != 0 ||
      (tokens > 1 && x_stride < K) || (channels > 1 && w_stride < K))
    return fail(SSM_ERR_INVALID, "linear_fp8: 8-bit rows must start at multiples of 16 bytes and not overlap");
  if (y.dtype != SSM_F32 && y.dtype != SSM_BF16) return fail(SSM_ERR_DTYPE, "linear_fp8: y dtype %lld unsupported", y.dtype);
  if (residual.ptr != nullptr && residual.dtype != y.dtype)
    return fail(SSM_ERR_DTYPE, "linear_fp8: the residual must have y's dtype");
  LinearParams p = {};
  const int tn = tile_tokens(tokens);
  if (!encode_rows8(&p.tw, w8, channels, K, w_stride, kRowsW) || !encode_rows8(&p.tx, x8, tokens, K, x_stride, tn))
    return fail(SSM_ERR_CUDA, "linear_fp8: the tensor maps could not be made");
  p.w_scale = w_scale;
  p.x_scale = x_scale;
  p.bias = bias;
  p.res = residual.ptr;
  p.rs = residual.batch_stride;
  p.y = const_cast<void*>(y.ptr);
  p.ys = y.batch_stride;
  p.tokens = (int)tokens;
  p.channels = (int)channels;
  p.blocks = (int)((K + kBlockK - 1) / kBlockK);
  p.silu = silu != 0;
  p.err = device_error_word();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = y.dtype == SSM_BF16 ? run_tokens<__nv_bfloat16>(p, tn, st) : run_tokens<float>(p, tn, st);
  return e == cudaSuccess ? SSM_OK : fail(SSM_ERR_CUDA, "linear_fp8 launch failed (error %lld)", (long long)e);
}

}  // extern "C"
