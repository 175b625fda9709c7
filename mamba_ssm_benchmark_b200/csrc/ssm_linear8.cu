// ssm_linear8.cu — products of 8-bit rows (e4m3, a float32 scale for every row) with everything behind them.
//
//   y[m, n] = act(x_scale[m] w_scale[n] sum_k x8[m, k] w8[n, k] + bias[n]) + residual[m, n]
//
// Two forms of one kernel.  Few tokens (or rows of y that are not aligned to 16 bytes): the weight's 128 rows are the M
// of tcgen05.mma (lanes of tensor memory), 16 to 256 tokens its N (columns), and 32 lanes store 32 neighbouring channels of
// a token.  More: 128 tokens are the M, 64 to 256 channels the N, and a lane stores 32 bytes of its token's row at a time (two
// bytes a lane at a time made the results, not the products, the bound: 16384 x 5120 x 2560 in 250 us whatever K).
// TMA brings 128-byte K blocks of both (128-byte swizzle; what lies past an edge is zero); a warp copies, a warp
// multiplies, eight warps read the accumulators of one tile while the next is multiplied.  Few tiles: the CTAs of a
// cluster take a part of K each and add their sums, in order, through distributed shared memory.
//
// 16384 x 5120 x 2560 with bias and residual: 163 us alone behind a cleared L2 (2.6 PFLOP/s, tensor pipe 77 % active), 196 to 207
// in a stream of calls, where the card's power decides.  Without them 156 and 179; so cuBLAS 171 and 182 with row scales, 164 and
// 154 with one scale.  64 x 2560 x 10240: 11.9 us for 26 MB of weights: prologue 1.5, two parts of K 3.0, their joining 2.8,
// barriers and the end 2 (clocks in the kernel).
// Wider joins (16 tokens, or 16 bytes a lane, at a time) were no faster.
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
  CUtensorMap ta, tb;                         // of the 128 rows (M) and of the columns (N)
  const float *w_scale, *x_scale, *bias;      // bias may be null
  const void* res;                            // null, or like y
  void* y;
  long long rs, ys;                           // row strides
  int tokens, channels, blocks;               // blocks of K
  int tiles_n, tiles;                         // tiles over the channels, and in all
  int silu;
  int wide;                                   // rows of y and res start at multiples of 32 bytes
  int* err;
};

constexpr int kRows = 128, kBlockK = 128;
constexpr int kOutWarps = 8, kLinThreads = 32 * (kOutWarps + 2);        // warps for results; one copies, one multiplies

template <int TN>
struct LinearForm {
  static constexpr int kStage = (kRows + TN) * kBlockK;
  // TN <= 64: two CTAs share an SM; above, one with as many stages as fit
  static constexpr int kStages = TN <= 32 ? 5 : TN == 64 ? 4 : TN == 128 ? 6 : 4;
  static constexpr uint32_t kCols = 2 * TN;
};
template <int TN>
struct LinearBars {
  uint64_t full[LinearForm<TN>::kStages], empty[LinearForm<TN>::kStages], acc_full[2], acc_empty[2];
  float scale[2][TN], bias[2][TN];            // of the columns, by accumulator
  uint32_t tmem;
};
template <int TN>
constexpr size_t linear_smem() { return (size_t)LinearForm<TN>::kStages * LinearForm<TN>::kStage + 1024 + sizeof(LinearBars<TN>); }

__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
                   smem_u32(dst)),
               "l"(map), "r"(c0), "r"(c1), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* map, int c0, int c1) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(map), "r"(c0), "r"(c1) : "memory");
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

__device__ __forceinline__ float2 act(const LinearParams& p, float2 v) {
  if (!p.silu) return v;
  return make_float2(v.x / (1.0f + __expf(-v.x)), v.y / (1.0f + __expf(-v.y)));
}
// 32 bytes, from or to rows that start at multiples of 16 or (wide) 32
__device__ __forceinline__ void load32(const void* src, bool wide, uint32_t (&w)[8]) {
  if (wide) {
    asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(src)
                 : "memory");
  } else {
    const uint4 a = static_cast<const uint4*>(src)[0], b = static_cast<const uint4*>(src)[1];
    w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
  }
}
__device__ __forceinline__ void store32(void* dst, bool wide, const uint32_t (&w)[8]) {
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                 "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  } else {
    static_cast<uint4*>(dst)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    static_cast<uint4*>(dst)[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

// 16 columns of this warp's 32 lanes on their way to v; they are there behind acc_wait.
__device__ __forceinline__ void acc_load(uint32_t addr, uint32_t (&v)[16]) {
  __syncwarp();
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void acc_wait(uint32_t (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]),
                 "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
               :
               : "memory");
}
// The values of 16 columns before the residual; scale and bias are the columns', `lane_scale` and `lane_bias` this lane's.
__device__ __forceinline__ void finish16(const LinearParams& p, const uint32_t (&v)[16], float lane_scale, float lane_bias,
                                         const float* scale, const float* bias, float2 (&r)[8]) {
  const float2 ls = bc2(lane_scale), lb = bc2(lane_bias);
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float4 s = *reinterpret_cast<const float4*>(scale + 2 * i);
    float4 b = make_float4(lb.x, lb.x, lb.x, lb.x);
    if (bias != nullptr) b = *reinterpret_cast<const float4*>(bias + 2 * i);
    r[i] = fma2(mul2(make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), ls), make_float2(s.x, s.y),
                make_float2(b.x, b.y));
    r[i + 1] = fma2(mul2(make_float2(__uint_as_float(v[2 * i + 2]), __uint_as_float(v[2 * i + 3])), ls), make_float2(s.z, s.w),
                    make_float2(b.z, b.w));
  }
  if (p.silu) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = act(p, r[i]);
  }
}

// Results of a tile whose lanes are tokens: this lane's token m, COLS channels from n0 on, 32 bytes of y at a time; the
// residuals of the next group are on their way while one is worked on, and so are the next accumulators.
template <int COLS, typename TY>
struct TokenRow {
  static constexpr int kVals = 32 / (int)sizeof(TY), kPer = 16 / kVals;           // values in 32 bytes, of these in 16 columns
  static constexpr int kGroup = COLS < 4 * kVals ? COLS : 4 * kVals, kLoads = kGroup / kVals;
  const LinearParams& p;
  const TY* res;
  TY* y;
  int left;                                   // channels of the row from n0 on, 0 past the last token
  uint32_t next[kLoads][8];
  __device__ TokenRow(const LinearParams& p_, int m, int n0) : p(p_) {
    left = m < p.tokens ? max(0, min(COLS, p.channels - n0)) : 0;
    res = p.res != nullptr && left > 0 ? static_cast<const TY*>(p.res) + m * p.rs + n0 : nullptr;
    y = static_cast<TY*>(p.y) + m * p.ys + n0;
    fetch(0);
  }
  __device__ __forceinline__ void fetch(int c) {
    if (res == nullptr) return;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int at = c + i * kVals;
      if (at + kVals <= left) {
        load32(res + at, p.wide, next[i]);
      } else if (at < left) {                 // the first half: rows are whole multiples of 16 bytes
        const uint4 q = *reinterpret_cast<const uint4*>(res + at);
        next[i][0] = q.x, next[i][1] = q.y, next[i][2] = q.z, next[i][3] = q.w;
      }
    }
  }
  __device__ __forceinline__ void finish(uint32_t acc, float x_scale, const float* w_scale, const float* bias) {
    uint32_t v[2][16];
    acc_load(acc, v[0]);
#pragma unroll
    for (int c0 = 0; c0 < COLS; c0 += kGroup) {
      uint32_t now[kLoads][8];
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) now[i][j] = next[i][j];
      if (c0 + kGroup < COLS) fetch(c0 + kGroup);
#pragma unroll
      for (int c = c0; c < c0 + kGroup; c += 16) {
        uint32_t(&a)[16] = v[c / 16 & 1];
        acc_wait(a);
        if (c + 16 < COLS) acc_load(acc + c + 16, v[c / 16 + 1 & 1]);
        float2 r[8];
        finish16(p, a, x_scale, 0.0f, w_scale + c, bias != nullptr ? bias + c : nullptr, r);
#pragma unroll
        for (int q = 0; q < kPer; ++q) {
          uint32_t(&old)[8] = now[(c - c0) / kVals + q];
          uint32_t w[8];
#pragma unroll
          for (int j = 0; j < kVals / 2; ++j) {
            float2 x = r[q * (kVals / 2) + j];
            if constexpr (sizeof(TY) == 2) {
              if (res != nullptr) x = add2(x, make_float2(lo_f32(old[j]), hi_f32(old[j])));
              w[j] = pack_bf16(x.x, x.y);
            } else {
              if (res != nullptr) x = add2(x, make_float2(__uint_as_float(old[2 * j]), __uint_as_float(old[2 * j + 1])));
              w[2 * j] = __float_as_uint(x.x);
              w[2 * j + 1] = __float_as_uint(x.y);
            }
          }
          const int at = c + q * kVals;
          if (at + kVals <= left)
            store32(y + at, p.wide, w);
          else if (at < left)
            *reinterpret_cast<uint4*>(y + at) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
  }
};

// Results of a tile whose lanes are channels: this lane's channel n, COLS tokens from m0 on, 16 at a time; 32 lanes store 32
// neighbours.  The next tokens' residuals are on their way.
template <int COLS, typename TY>
__device__ __forceinline__ void finish_channel(const LinearParams& p, uint32_t acc, int m0, int n, const float* x_scale,
                                               float w_scale, float bias) {
  const int left = n < p.channels ? min(COLS, p.tokens - m0) : 0;
  const TY* rp = static_cast<const TY*>(p.res) + (long long)m0 * p.rs + n;
  TY* yp = static_cast<TY*>(p.y) + (long long)m0 * p.ys + n;
  const bool adds = p.res != nullptr;
  TY next[16];
  auto fetch = [&](int c) {
#pragma unroll
    for (int i = 0; i < 16; ++i, rp += p.rs) next[i] = adds && c + i < left ? *rp : from_f32<TY>(0.0f);
  };
  fetch(0);
  for (int c = 0; c < COLS; c += 16) {
    uint32_t v[16];
    float2 r[8];
    acc_load(acc + c, v);
    acc_wait(v);
    finish16(p, v, w_scale, bias, x_scale + c, nullptr, r);
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = add2(r[i], make_float2(to_f32(next[2 * i]), to_f32(next[2 * i + 1])));
    if (c + 16 < COLS) fetch(c + 16);
#pragma unroll
    for (int i = 0; i < 16; ++i, yp += p.ys)
      if (c + i < left) *yp = from_f32<TY>(i & 1 ? r[i / 2].y : r[i / 2].x);
  }
}

// TOKENS: the lanes are tokens and the columns channels, else the other way about.  SPLIT: a cluster takes one tile, its
// CTAs a part of K each.
template <int TN, typename TY, bool TOKENS, bool SPLIT>
__global__ void __launch_bounds__(kLinThreads, TN <= 64 ? 2 : 1) linear_e4m3(const __grid_constant__ LinearParams p, int parts) {
  static_assert(!SPLIT || TN <= 64, "parts of K are for few tiles, which are narrow");
  using Form = LinearForm<TN>;
  constexpr int kStages = Form::kStages;
  extern __shared__ unsigned char raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  auto& bar = *reinterpret_cast<LinearBars<TN>*>(smem + (size_t)kStages * Form::kStage);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = SPLIT ? (int)cluster_rank() : 0;
  const int first = SPLIT ? (int)blockIdx.x / parts : (int)blockIdx.x, step = SPLIT ? p.tiles : (int)gridDim.x;
  const int k0 = SPLIT ? (int)((long long)p.blocks * rank / parts) : 0;
  const int k1 = SPLIT ? (int)((long long)p.blocks * (rank + 1) / parts) : p.blocks;
  // What the first tile reads of the weight goes to L2 while the kernel before still runs (L2 is where all writes meet, so a
  // weight that this kernel writes is not read stale): a layer as below with 64 tokens takes 24.3 us for 27.3, with 16 tokens
  // 18.3 for 21.0, with one 18.8 for 19.7.  With tokens in the lanes it gained 1 % of a layer of 128 and lost as much of one
  // of 512.
  if (!TOKENS && warp == kOutWarps) {
    const int row = first % p.tiles_n * kRows;
    for (int k = k0 + lane; k < k1; k += 32) tma_prefetch_2d(&p.ta, k * kBlockK, row);
    if (row + lane * 32 < p.channels && lane < kRows / 32) {
      prefetch_l2(p.w_scale + row + lane * 32);
      if (p.bias != nullptr) prefetch_l2(p.bias + row + lane * 32);
    }
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&bar.full[i], 1);
      mbar_init(&bar.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar.acc_full[i], 1);
      mbar_init(&bar.acc_empty[i], kOutWarps);
    }
    fence_mbar_init();
  }
  if (warp == kOutWarps + 1) tc_alloc(&bar.tmem, Form::kCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = __shfl_sync(0xffffffffu, bar.tmem, 0);
  // What is above needs no memory of others.  The next kernel may come as soon as this one's CTAs are all there: a layer of norm,
  // product, quantisation and product (2560 channels, one token, graph) takes 23.3 us without early launches, 21.3 when the
  // products let the next one in at their end and 19.8 so; only products of 64 tokens with nothing between them lose (10.7
  // against 12.3 us: the next one's CTAs take places beside this one's and share the SMs unevenly).
  pdl_launch_dependents();
  pdl_wait();
  constexpr int kTileM = TOKENS ? kRows : TN, kTileN = TOKENS ? TN : kRows;      // tokens and channels of a tile
  auto tile_m = [&](int t) { return t / p.tiles_n * kTileM; };
  auto tile_n = [&](int t) { return t % p.tiles_n * kTileN; };
  Wait wait{p.err};
  if (warp == kOutWarps) {                               // copies
    if (lane == 0) {
      int st = 0, par = 1;
      for (int t = first; t < p.tiles && !wait.dead; t += step) {
        const int a0 = TOKENS ? tile_m(t) : tile_n(t), b0 = TOKENS ? tile_n(t) : tile_m(t);
        for (int k = k0; k < k1; ++k) {
          wait(&bar.empty[st], par);
          if (wait.dead) break;
          unsigned char* at = smem + (size_t)st * Form::kStage;
          mbar_arrive_expect_tx(&bar.full[st], Form::kStage);
          tma_load_2d(at, &p.ta, &bar.full[st], k * kBlockK, a0);
          tma_load_2d(at + kRows * kBlockK, &p.tb, &bar.full[st], k * kBlockK, b0);
          if (++st == kStages) st = 0, par ^= 1;
        }
      }
    }
    __syncwarp();
  } else if (warp == kOutWarps + 1) {                    // products
    const uint32_t issue = lane == 0;
    // fp32 accumulators, both operands e4m3 and read along their rows, M = 128
    const uint32_t idesc = 1u << 4 | (uint32_t)(TN / 8) << 17 | (kRows / 16u) << 24;
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
        const uint32_t a = tc_desc(smem_u32(smem + (size_t)st * Form::kStage), 16), b = a + kRows * kBlockK / 16;
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
    // a warp reads the 32 lanes of its number modulo 4; the second four have the second half of the columns
    constexpr int kCols = TN > 16 ? TN / 2 : TN;
    const uint32_t my = tm + ((uint32_t)(32 * (warp & 3)) << 16);
    const int row = 32 * (warp & 3) + lane, half = (warp >> 2) * kCols;
    const bool works = half < TN;
    int buf = 0, bpar = 0;
    for (int t = first; t < p.tiles; t += step) {        // to the end also after a wait that gave up: the warps meet
      const int m0 = tile_m(t), n0 = tile_n(t);
      if constexpr (SPLIT) {
        wait(&bar.acc_full[buf], bpar);
        wait.dead = __any_sync(0xffffffffu, wait.dead);
        tc_fence_after();
        // over the stages, whose products are done: [token][channel], where lanes are tokens in rows of TN + 1, which keeps
        // their banks apart
        float* part = reinterpret_cast<float*>(smem);
        if (works) {
#pragma unroll
          for (int c = 0; c < kCols; c += 16) {
            float v[16];
            tc_load_f32(my + buf * TN + half + c, v);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int col = half + c + i;
              part[TOKENS ? row * (TN + 1) + col : col * kRows + row] = wait.dead ? quiet_nan() : v[i];
            }
          }
        }
        tc_fence_before();
      } else {
        // The columns' scales and biases; a warp is at most one barrier ahead of those that read the other buffer.
        for (int c = threadIdx.x; c < TN; c += 32 * kOutWarps) {
          const int at = (TOKENS ? n0 : m0) + c;
          const bool in = at < (TOKENS ? p.channels : p.tokens);
          bar.scale[buf][c] = in ? (TOKENS ? p.w_scale : p.x_scale)[at] : 0.0f;
          if (TOKENS && p.bias != nullptr) bar.bias[buf][c] = in ? p.bias[at] : 0.0f;
        }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kOutWarps) : "memory");
        if constexpr (TOKENS) {
          TokenRow<kCols, TY> out(p, m0 + row, n0 + half);
          const float xs = m0 + row < p.tokens ? p.x_scale[m0 + row] : 0.0f;
          wait(&bar.acc_full[buf], bpar);
          wait.dead = __any_sync(0xffffffffu, wait.dead);
          tc_fence_after();
          const float* bias = p.bias != nullptr ? bar.bias[buf] + half : nullptr;
          if (!wait.dead) out.finish(my + buf * TN + half, xs, bar.scale[buf] + half, bias);
        } else {
          const int n = n0 + row;
          const float ws = n < p.channels ? p.w_scale[n] : 0.0f, bias = n < p.channels && p.bias != nullptr ? p.bias[n] : 0.0f;
          wait(&bar.acc_full[buf], bpar);
          wait.dead = __any_sync(0xffffffffu, wait.dead);
          tc_fence_after();
          if (!wait.dead && works)
            finish_channel<kCols, TY>(p, my + buf * TN + half, m0 + half, n, bar.scale[buf] + half, ws, bias);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) tc_arrive(&bar.acc_empty[buf]);
      }
      if (++buf == 2) buf = 0, bpar ^= 1;
    }
    __syncwarp();
  }
  if constexpr (SPLIT) {
    __syncwarp();
    cluster_arrive_wait();
    // this CTA's tokens; a warp takes kJoin of them and 32 channels at a time, so that as many loads are on their way
    constexpr int kPitch = TOKENS ? TN + 1 : kRows, kJoin = TOKENS ? 8 : TN / 8;
    const int own = kTileM / parts, m0 = tile_m(first), n0 = tile_n(first);
    for (int item = warp; item < own / kJoin * (kTileN / 32); item += kLinThreads / 32) {
      const int c0 = rank * own + item / (kTileN / 32) * kJoin, col = item % (kTileN / 32) * 32 + lane, n = n0 + col;
      if (n >= p.channels || m0 + c0 >= p.tokens) continue;
      const float ws = p.w_scale[n], bias = p.bias != nullptr ? p.bias[n] : 0.0f;
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
        for (int i = 0; i < kJoin; ++i)
          v[i] += peer_load(smem_u32(smem) + ((c0 + i) * kPitch + col) * 4, q);
      }
#pragma unroll
      for (int i = 0; i < kJoin; i += 2) {
        const float2 r = act(p, fma2(mul2(make_float2(v[i], v[i + 1]), make_float2(xs[i], xs[i + 1])), bc2(ws), bc2(bias)));
        TY* y = static_cast<TY*>(p.y) + (m0 + c0 + i) * p.ys + n;
        if (m0 + c0 + i < p.tokens) y[0] = from_f32<TY>(r.x + res[i]);
        if (m0 + c0 + i + 1 < p.tokens) y[p.ys] = from_f32<TY>(r.y + res[i + 1]);
      }
    }
    __syncwarp();
    cluster_arrive_wait();                               // peers read this CTA's sums until here
  }
  wait.drain();
  __syncthreads();
  if (warp == kOutWarps + 1) tc_free(tm, Form::kCols);
}

// ---- host -----------------------------------------------------------------------------------
int fail(int code, const char* fmt, long long a = 0, long long b = 0) {
  char msg[256];
  snprintf(msg, sizeof(msg), fmt, a, b);
  return report_error(code, msg);
}
int ceil_div(int a, int b) { return (a + b - 1) / b; }

template <int TN, typename TY, bool TOKENS, bool SPLIT>
cudaError_t launch(const LinearParams& p, int ctas, int parts, cudaStream_t st) {
  constexpr auto kern = linear_e4m3<TN, TY, TOKENS, SPLIT>;
  ctas_per_sm<kern>(kLinThreads, linear_smem<TN>());
  return launch_pdl_cluster(kern, (unsigned)ctas, kLinThreads, SPLIT ? (unsigned)parts : 0, linear_smem<TN>(), st, p, parts);
}

constexpr int room(int tn) { return 148 * (tn <= 64 ? 2 : 1); }         // CTAs that run at once
template <int TN, typename TY, bool TOKENS>
cudaError_t run(LinearParams& p, cudaStream_t st) {
  p.tiles_n = ceil_div(p.channels, TOKENS ? TN : kRows);
  p.tiles = p.tiles_n * ceil_div(p.tokens, TOKENS ? kRows : TN);
  // wider tiles are taken where there are 148 of them or more: one to an SM, which leaves no room for parts of K
  if constexpr (TN <= 64) {
    int parts = 1;
    while (parts < 8 && p.tiles * parts * 2 <= room(TN) && parts * 2 <= p.blocks) parts *= 2;
    if (parts > 1) return launch<TN, TY, TOKENS, true>(p, p.tiles * parts, parts, st);
  }
  return launch<TN, TY, TOKENS, false>(p, std::min(p.tiles, room(TN)), 1, st);
}
template <typename TY>
cudaError_t run_form(LinearParams& p, bool tokens, int tn, cudaStream_t st) {
  if (tokens) {
    if (tn == 64) return run<64, TY, true>(p, st);
    if (tn == 128) return run<128, TY, true>(p, st);
    return run<256, TY, true>(p, st);
  }
  if (tn == 16) return run<16, TY, false>(p, st);
  if (tn == 32) return run<32, TY, false>(p, st);
  if (tn == 64) return run<64, TY, false>(p, st);
  if (tn == 128) return run<128, TY, false>(p, st);
  return run<256, TY, false>(p, st);
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
  const int es = y.dtype == SSM_BF16 ? 2 : 4;
  auto aligned = [&](int n) {
    auto fits = [&](const ssm_view& v) { return reinterpret_cast<uintptr_t>(v.ptr) % n == 0 && v.batch_stride * es % n == 0; };
    return fits(y) && (residual.ptr == nullptr || fits(residual));
  };
  // Columns of a tile: the fewest that hold the tokens, where these are few (or y's rows do not allow the other form); else as
  // many channels as leave every SM a tile.
  const bool by_token = tokens > 64 && aligned(16) && channels * es % 16 == 0;
  const int64_t cols = by_token ? channels : tokens, lanes = by_token ? tokens : channels;
  int tn = 16;
  if (cols > 64) {
    tn = 256;
    while (tn > 64 && (cols + tn - 1) / tn * ((lanes + kRows - 1) / kRows) < 148) tn /= 2;
  } else {
    while (tn < cols) tn *= 2;
  }
  if (by_token && tn < 64) tn = 64;
  p.wide = aligned(32);
  CUtensorMap &mx = by_token ? p.ta : p.tb, &mw = by_token ? p.tb : p.ta;
  if (!encode_rows8(&mx, x8, tokens, K, x_stride, by_token ? kRows : tn) ||
      !encode_rows8(&mw, w8, channels, K, w_stride, by_token ? tn : kRows))
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
  const cudaError_t e = es == 2 ? run_form<__nv_bfloat16>(p, by_token, tn, st) : run_form<float>(p, by_token, tn, st);
  return e == cudaSuccess ? SSM_OK : fail(SSM_ERR_CUDA, "linear_fp8 launch failed (error %lld)", (long long)e);
}

}  // extern "C"
