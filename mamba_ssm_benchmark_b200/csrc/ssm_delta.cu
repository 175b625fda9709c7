// ssm_delta.cu — the gated delta rule: chunked forward and backward, one-token state update.
// The formulas are in ssm_delta.cuh.  Forward: delta_prep (everything that does not need the state, all
// chunks at once), delta_fwd (the state from chunk to chunk, and the output).  Backward: delta_prep,
// delta_bwd_chain (the state's gradient from the last chunk to the first), delta_bwd_chunk (all other
// gradients, all chunks at once), delta_sum_heads (query and key gradients over the value heads that
// share a key head).
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdio>
#include <cstring>

#include "ssm_b200.h"
#include "ssm_delta.cuh"
#include "ssm_vec.cuh"

namespace ssm {
int report_error(int code, const char* msg);
int* device_error_word();
}  // namespace ssm

namespace {

using namespace ssm;

constexpr int kPitch = kC + 4;

// ================================================================================================
// Chunk preparation: one CTA of four warps per (chunk, value head, batch).
// ================================================================================================
// 8 columns of a row as float; zero outside.
template <typename T>
__device__ __forceinline__ void load8(const T* row, int c0, int width, bool vec, float (&x)[8]) {
  if (vec && c0 + 8 <= width) {
    if constexpr (sizeof(T) == 2) {
      vec_load<T, 8>(row + c0, x);
    } else {
      float a[4], b[4];
      load4(row + c0, a);
      load4(row + c0 + 4, b);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = a[i];
        x[4 + i] = b[i];
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = c0 + i < width ? to_f32(row[c0 + i]) : 0.0f;
  }
}

// Splits 8 values into NP pieces and writes 16 bytes of each at `off` of the tiles `stride` apart.
template <int NP>
__device__ __forceinline__ void put_pieces(const float (&x)[8], __nv_bfloat16* shared, __nv_bfloat16* global, int off,
                                           int stride) {
  uint32_t p[4][NP];
#pragma unroll
  for (int i = 0; i < 4; ++i) split<NP>(x[2 * i], x[2 * i + 1], p[i]);
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const uint4 w = make_uint4(p[0][i], p[1][i], p[2][i], p[3][i]);
    if (shared != nullptr) *reinterpret_cast<uint4*>(shared + i * stride + off) = w;
    if (global != nullptr) *reinterpret_cast<uint4*>(global + i * stride + off) = w;
  }
}

__device__ __forceinline__ bool rows_aligned16(const Heads& h, int es) {
  return ((reinterpret_cast<uintptr_t>(h.ptr) | (uintptr_t)(h.sb * es) | (uintptr_t)(h.sl * es) |
           (uintptr_t)(h.sh * es)) & 15) == 0;
}

template <typename T, int NP, int DKP>
struct PrepSmem {
  __nv_bfloat16 k[NP][kC * DKP], q[NP][kC * DKP];
  float A[kC][kPitch], T_[kC][kPitch], P[kC][kPitch], tmp[32][36];
  float gh[kC], gl[kC], beta[kC];
};

template <typename T, int NP, int DKP>
__global__ void __launch_bounds__(128) delta_prep(const DeltaParams p) {
  extern __shared__ __align__(128) unsigned char smem_raw[];
  auto& s = *reinterpret_cast<PrepSmem<T, NP, DKP>*>(smem_raw);
  const int ch = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int t0 = ch * kC, rows = min(kC, p.L - t0), hk = h / p.group;
  const size_t at = ((size_t)b * p.Hv + h) * p.n + ch;
  const size_t atk = ((size_t)b * p.Hk + hk) * p.n + ch;

  // q and k in pieces: into shared memory and, once per key head, into the tiles the chain kernels load
  {
    const bool writer = h % p.group == 0;
    const T* kb = static_cast<const T*>(p.k.ptr) + b * p.k.sb + t0 * p.k.sl + hk * p.k.sh;
    const T* qb = static_cast<const T*>(p.q.ptr) + b * p.q.sb + t0 * p.q.sl + hk * p.q.sh;
    const bool kv = rows_aligned16(p.k, sizeof(T)), qv = rows_aligned16(p.q, sizeof(T));
    __nv_bfloat16* kg = writer ? p.kimg + atk * (NP * kC * DKP) : nullptr;
    __nv_bfloat16* qg = writer ? p.qimg + atk * (NP * kC * DKP) : nullptr;
    for (int e = tid; e < kC * DKP / 8; e += 128) {
      const int r = e / (DKP / 8), grp = e % (DKP / 8), width = r < rows ? p.dkw : 0;
      float x[8], y[8];
      load8<T>(kb + (long long)r * p.k.sl, grp * 8, width, kv, x);
      load8<T>(qb + (long long)r * p.q.sl, grp * 8, width, qv, y);
      const int off = tile_off<DKP>(r, grp);
      put_pieces<NP>(x, s.k[0], kg, off, kC * DKP);
      put_pieces<NP>(y, s.q[0], qg, off, kC * DKP);
    }
  }
  // running sums of g.  In double and kept as two floats: differences of neighbours stay exact to fp32
  // also behind a position that resets the state.  exp(-1000) is 0, so -inf can be taken as -1000.
  if (warp == 0) {
    double acc[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = 2 * lane + i;
      float g = r < rows ? p.g[b * p.gsb + (t0 + r) * p.gsl + h] : 0.0f;
      g = g < -1000.0f ? -1000.0f : g;
      acc[i] = (double)g * 1.4426950408889634;
      s.beta[r] = r < rows ? p.beta[b * p.bsb + (t0 + r) * p.bsl + h] : 0.0f;
    }
    acc[1] += acc[0];
    double run = acc[1];
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, run, m);
      if (lane >= m) run += up;
    }
    const double total = __shfl_sync(0xffffffffu, run, 31);
    const double G[2] = {run - (acc[1] - acc[0]), run};
    float* vec = p.vec + at * kVec;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = 2 * lane + i;
      const float hi = (float)G[i], lo = (float)(G[i] - (double)hi);
      s.gh[r] = hi;
      s.gl[r] = lo;
      vec[r] = exp2f((float)G[i]);
      vec[kC + r] = exp2f((float)(total - G[i]));
      vec[2 * kC + r] = s.beta[r];
      vec[3 * kC + r] = hi;
      vec[4 * kC + r] = lo;
    }
  }
  for (int e = tid; e < kC * kPitch; e += 128) (&s.T_[0][0])[e] = 0.0f;
  __syncthreads();

  // k.k and q.k of the warp's 16 rows against the columns up to its own
  {
    float kk[kC / 8][4], qk[kC / 8][4];
    zero(kk);
    zero(qk);
    const uint32_t sk = smem_u32(s.k[0]), sq = smem_u32(s.q[0]);
#pragma unroll 2
    for (int kb = 0; kb < DKP / 16; ++kb) {
      uint32_t ak[NP][4], aq[NP][4];
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        load_a<DKP>(ak[i], sk + i * (kC * DKP * 2), 16 * warp, kb, lane);
        load_a<DKP>(aq[i], sq + i * (kC * DKP * 2), 16 * warp, kb, lane);
      }
#pragma unroll
      for (int jp = 0; jp < kC / 16; ++jp) {
        if (jp > warp) break;
#pragma unroll
        for (int pb = 0; pb < NP; ++pb) {
          uint32_t bf[4];
          load_b<DKP>(bf, sk + pb * (kC * DKP * 2), 2 * jp, kb, lane);
          mma_pieces<NP, 2>(kk[2 * jp], kk[2 * jp + 1], ak, bf, pb);
          mma_pieces<NP, 2>(qk[2 * jp], qk[2 * jp + 1], aq, bf, pb);
        }
      }
    }
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int j = 0; j < kC / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = 16 * warp + g + 8 * (e >> 1), c = 8 * j + 2 * t + (e & 1);
        const float d = i >= c ? ex2((s.gh[i] - s.gh[c]) + (s.gl[i] - s.gl[c])) : 0.0f;
        s.A[i][c] = i > c ? s.beta[i] * (d * kk[j][e]) : 0.0f;
        s.P[i][c] = i >= c ? p.scale * (d * qk[j][e]) : 0.0f;
      }
  }
  __syncthreads();

  // T = (I + A)^-1 by forward substitution: the diagonal 16 x 16 blocks, then the blocks below them
  // from the blocks beside: T21 = -T22 A21 T11.
  if (lane < 16) {
    const int r0 = 16 * warp;
    float t[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v = i == lane ? 1.0f : 0.0f;
#pragma unroll
      for (int m = 0; m < i; ++m) v = fmaf(-s.A[r0 + i][r0 + m], t[m], v);
      t[i] = v;
      s.T_[r0 + i][r0 + lane] = v;
    }
  }
  __syncthreads();
  {
    const int pr = 32 * (tid >> 6), r = (tid & 63) >> 2, c = 4 * (tid & 3);
    float y[4] = {0.f, 0.f, 0.f, 0.f};
    for (int m = 0; m < 16; ++m) {
      const float a = s.A[pr + 16 + r][pr + m];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = fmaf(a, s.T_[pr + m][pr + c + e], y[e]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) s.tmp[r][(pr >> 1) + c + e] = y[e];
  }
  __syncthreads();
  {
    const int pr = 32 * (tid >> 6), r = (tid & 63) >> 2, c = 4 * (tid & 3);
    float y[4] = {0.f, 0.f, 0.f, 0.f};
    for (int m = 0; m < 16; ++m) {
      const float a = s.T_[pr + 16 + r][pr + 16 + m];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = fmaf(-a, s.tmp[m][(pr >> 1) + c + e], y[e]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) s.T_[pr + 16 + r][pr + c + e] = y[e];
  }
  __syncthreads();
  {
    const int r = tid >> 2, c = 8 * (tid & 3);
    float y[8] = {};
    for (int m = 0; m < 32; ++m) {
      const float a = s.A[32 + r][m];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = fmaf(a, s.T_[m][c + e], y[e]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) s.tmp[r][c + e] = y[e];
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = 0.0f;
    for (int m = 0; m < 32; ++m) {
      const float a = s.T_[32 + r][32 + m];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = fmaf(-a, s.tmp[m][c + e], y[e]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) s.T_[32 + r][c + e] = y[e];
  }
  __syncthreads();
  for (int e = tid; e < kC * kC / 8; e += 128) {
    const int r = e / (kC / 8), grp = e % (kC / 8), off = tile_off<kC>(r, grp);
    float x[8], y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = s.T_[r][grp * 8 + i];
      y[i] = s.P[r][grp * 8 + i];
    }
    put_pieces<3>(x, nullptr, p.timg + at * (3 * kTri), off, kTri);
    put_pieces<3>(y, nullptr, p.pimg + at * (3 * kTri), off, kTri);
  }
}

// ================================================================================================
// The chain kernels' shared memory: the tiles of one chunk, loaded by bulk copies.
// ================================================================================================
template <int NP, int DKP, int PP>     // PP: pieces of P
struct alignas(128) ChainStage {
  __nv_bfloat16 k[NP][kC * DKP], q[NP][kC * DKP];
  __nv_bfloat16 t[3][kTri], pm[PP][kTri];
  float vec[kVec];
};
template <int NP, int DKP, int PP>
constexpr int chain_stages() {
  return 2 * sizeof(ChainStage<NP, DKP, PP>) + 256 <= 227 * 1024 ? 2 : 1;
}
template <int NP, int DKP, int PP>
constexpr size_t chain_smem() {
  return chain_stages<NP, DKP, PP>() * sizeof(ChainStage<NP, DKP, PP>) + 128;
}

template <int NP, int DKP, int PP>
__device__ __forceinline__ void chain_load(ChainStage<NP, DKP, PP>& s, const DeltaParams& p, int b, int h, int ch,
                                           uint64_t* bar) {
  const size_t at = ((size_t)b * p.Hv + h) * p.n + ch;
  const size_t atk = ((size_t)b * p.Hk + h / p.group) * p.n + ch;
  mbar_arrive_expect_tx(bar, sizeof(s.k) + sizeof(s.q) + sizeof(s.t) + sizeof(s.pm) + sizeof(s.vec));
  bulk_load(s.k, p.kimg + atk * (NP * kC * DKP), sizeof(s.k), bar);
  bulk_load(s.q, p.qimg + atk * (NP * kC * DKP), sizeof(s.q), bar);
  bulk_load(s.t, p.timg + at * (3 * kTri), sizeof(s.t), bar);
  bulk_load(s.pm, p.pimg + at * (3 * kTri), sizeof(s.pm), bar);
  bulk_load(s.vec, p.vec + at * kVec, sizeof(s.vec), bar);
}

// The state (dk, dv) of a head in global memory from / to the warp's accumulators of S^T.
template <int NT>
__device__ __forceinline__ void state_load(const float* base, int dk, int dv, int d0, int lane, float (&S)[NT][4]) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int k = 8 * j + 2 * t + (e & 1), d = d0 + g + 8 * (e >> 1);
      S[j][e] = base != nullptr && k < dk && d < dv ? base[(size_t)k * dv + d] : 0.0f;
    }
}
template <int NT>
__device__ __forceinline__ void state_store(float* base, int dk, int dv, int d0, int lane, const float (&S)[NT][4]) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int k = 8 * j + 2 * t + (e & 1), d = d0 + g + 8 * (e >> 1);
      if (k < dk && d < dv) base[(size_t)k * dv + d] = S[j][e];
    }
}

// R^T (16 x kC) = M^T-side product with a triangular kC x kC tile: D[.][i] += sum_k a[.][k] L[i][k] (TR false,
// L lower: tiles i >= k) or D[.][j] += sum_i a[.][i] L[i][j] (TR true: tiles j <= i).
template <int NA, int NB, int MAXI, bool TR>
__device__ __forceinline__ void tri_product(float (&d)[kC / 8][4], const float (&a)[kC / 8][4], uint32_t tile, int lane) {
#pragma unroll
  for (int kb = 0; kb < kC / 16; ++kb) {
    uint32_t af[NA][4];
    acc_to_a<NA>(a, kb, af);
#pragma unroll
    for (int jp = 0; jp < kC / 16; ++jp) {
      if (TR ? jp > kb : jp < kb) continue;
#pragma unroll
      for (int pb = 0; pb < NB; ++pb) {
        uint32_t bf[4];
        if (TR) load_bt<kC>(bf, tile + pb * (kTri * 2), 2 * jp, kb, lane);
        else load_b<kC>(bf, tile + pb * (kTri * 2), 2 * jp, kb, lane);
        mma_pieces<NA, MAXI>(d[2 * jp], d[2 * jp + 1], af, bf, pb);
      }
    }
  }
}

// S <- decay S + (a [.][c]) (tile [c][dk]) over kC positions.  The sum over the chunk is formed on its
// own and added once, rounded to nearest: the tensor cores' accumulation truncates, and a state that
// they accumulated over hundreds of chunks would drift.
template <int NP, int DKP>
__device__ __forceinline__ void state_add(float (&S)[DKP / 8][4], float decay, float sign, const float (&a)[kC / 8][4],
                                          uint32_t tile, int lane) {
  uint32_t af[kC / 16][3][4];
#pragma unroll
  for (int kb = 0; kb < kC / 16; ++kb) acc_to_a<3>(a, kb, af[kb]);
#pragma unroll
  for (int jp = 0; jp < DKP / 16; ++jp) {
    float d[2][4];
    zero(d);
#pragma unroll
    for (int kb = 0; kb < kC / 16; ++kb)
#pragma unroll
      for (int pb = 0; pb < NP; ++pb) {
        uint32_t bf[4];
        load_bt<DKP>(bf, tile + pb * (kC * DKP * 2), 2 * jp, kb, lane);
        mma_pieces<3, 2>(d[0], d[1], af[kb], bf, pb);
      }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) S[2 * jp + h][e] = fmaf(decay, S[2 * jp + h][e], sign * d[h][e]);
  }
}

// ================================================================================================
// Forward chain: a warp carries 16 value channels of one head's state through all chunks.
// ================================================================================================
template <typename T, int NP, int DKP, bool SAVE>
__global__ void __launch_bounds__(256) delta_fwd(const __grid_constant__ DeltaParams p) {
  constexpr int PP = NP == 1 ? 2 : 3;
  using Stage = ChainStage<NP, DKP, PP>;
  constexpr int kStages = chain_stages<NP, DKP, PP>();
  extern __shared__ __align__(128) unsigned char smem_raw[];
  Stage* stage = reinterpret_cast<Stage*>(smem_raw);
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem_raw + kStages * sizeof(Stage));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, t = lane & 3;
  const int h = blockIdx.y, b = blockIdx.z;
  const int d0 = 16 * (blockIdx.x * (blockDim.x >> 5) + warp), cols = p.dvw - d0;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&bar[i], 1);
    fence_mbar_init();
    for (int i = 0; i < kStages && i < p.n; ++i) chain_load(stage[i], p, b, h, i, &bar[i]);
  }
  const size_t head = (size_t)b * p.Hv + h;
  float S[DKP / 8][4];
  state_load(p.h0 != nullptr ? p.h0 + head * p.dkw * p.dvw : nullptr, p.dkw, p.dvw, d0, lane, S);
  __syncthreads();
  for (int ch = 0; ch < p.n; ++ch) {
    const int st = ch % kStages;
    const Stage& s = stage[st];
    const int rows = min(kC, p.L - ch * kC);
    const long long t0 = (long long)ch * kC;
    mbar_wait(&bar[st], (ch / kStages) & 1, p.err);
    if (cols > 0) {
      float V[kC / 8][4], X[kC / 8][4], O[kC / 8][4];
      load_vt(static_cast<const T*>(p.v.ptr) + b * p.v.sb + t0 * p.v.sl + h * p.v.sh + d0, p.v.sl, rows, cols, lane, V);
      if (SAVE) store_acc(p.states + ((head * p.n + ch) * p.dvp + d0) * DKP, DKP, lane, S);
      // K S and Q S (transposed)
      zero(X);
      zero(O);
      const uint32_t sk = smem_u32(s.k[0]), sq = smem_u32(s.q[0]);
#pragma unroll
      for (int kb = 0; kb < DKP / 16; ++kb) {
        uint32_t a[3][4];
        acc_to_a<3>(S, kb, a);
#pragma unroll
        for (int jp = 0; jp < kC / 16; ++jp)
#pragma unroll
          for (int pb = 0; pb < NP; ++pb) {
            uint32_t bf[4];
            load_b<DKP>(bf, sk + pb * (kC * DKP * 2), 2 * jp, kb, lane);
            mma_pieces<3, 2>(X[2 * jp], X[2 * jp + 1], a, bf, pb);
            load_b<DKP>(bf, sq + pb * (kC * DKP * 2), 2 * jp, kb, lane);
            mma_pieces<3, NP == 1 ? 1 : 2>(O[2 * jp], O[2 * jp + 1], a, bf, pb);   // bf16 o: 16 bits of S
          }
      }
#pragma unroll
      for (int j = 0; j < kC / 8; ++j) {
        const float2 eg = *reinterpret_cast<const float2*>(s.vec + 8 * j + 2 * t);
        const float2 be = *reinterpret_cast<const float2*>(s.vec + 2 * kC + 8 * j + 2 * t);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float eg_ = e & 1 ? eg.y : eg.x;
          X[j][e] = (e & 1 ? be.y : be.x) * fmaf(-eg_, X[j][e], V[j][e]);
          O[j][e] *= p.scale * eg_;
        }
      }
      float U[kC / 8][4];
      zero(U);
      tri_product<3, 3, 2, false>(U, X, smem_u32(s.t[0]), lane);
      if (SAVE) store_acc(p.us + ((head * p.n + ch) * p.dvp + d0) * kC, kC, lane, U);
      tri_product<PP, PP, PP - 1, false>(O, U, smem_u32(s.pm[0]), lane);
      store_vt(static_cast<T*>(const_cast<void*>(p.o.ptr)) + b * p.o.sb + t0 * p.o.sl + h * p.o.sh + d0, p.o.sl, rows,
               cols, lane, O);
#pragma unroll
      for (int j = 0; j < kC / 8; ++j) {
        const float2 la = *reinterpret_cast<const float2*>(s.vec + kC + 8 * j + 2 * t);
#pragma unroll
        for (int e = 0; e < 4; ++e) U[j][e] *= e & 1 ? la.y : la.x;
      }
      state_add<NP, DKP>(S, s.vec[kC - 1], 1.0f, U, sk, lane);
    }
    __syncthreads();
    if (threadIdx.x == 0 && ch + kStages < p.n) chain_load(stage[st], p, b, h, ch + kStages, &bar[st]);
  }
  if (cols > 0 && p.last != nullptr) state_store(p.last + head * p.dkw * p.dvw, p.dkw, p.dvw, d0, lane, S);
}

// ================================================================================================
// Backward chain, chunks in reverse, with dS' the gradient of the state leaving the chunk:
//   Y = e^(G_last - G) K dS' + P^T dO,  dX = T^T Y,  dV = beta dX
//   dS = e^G_last dS' + (scale e^G Q)^T dO - (beta e^G K)^T dX
// ================================================================================================
template <typename T, int NP, int DKP>
__global__ void __launch_bounds__(256) delta_bwd_chain(const __grid_constant__ DeltaParams p) {
  using Stage = ChainStage<NP, DKP, 3>;
  constexpr int kStages = chain_stages<NP, DKP, 3>();
  extern __shared__ __align__(128) unsigned char smem_raw[];
  Stage* stage = reinterpret_cast<Stage*>(smem_raw);
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem_raw + kStages * sizeof(Stage));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, t = lane & 3;
  const int h = blockIdx.y, b = blockIdx.z;
  const int d0 = 16 * (blockIdx.x * (blockDim.x >> 5) + warp), cols = p.dvw - d0;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&bar[i], 1);
    fence_mbar_init();
    for (int i = 0; i < kStages && i < p.n; ++i) chain_load(stage[i], p, b, h, p.n - 1 - i, &bar[i]);
  }
  const size_t head = (size_t)b * p.Hv + h;
  float S[DKP / 8][4];
  state_load(p.h0 != nullptr ? p.h0 + head * p.dkw * p.dvw : nullptr, p.dkw, p.dvw, d0, lane, S);
  __syncthreads();
  for (int it = 0; it < p.n; ++it) {
    const int ch = p.n - 1 - it, st = it % kStages;
    const Stage& s = stage[st];
    const int rows = min(kC, p.L - ch * kC);
    const long long t0 = (long long)ch * kC;
    mbar_wait(&bar[st], (it / kStages) & 1, p.err);
    if (cols > 0) {
      float dO[kC / 8][4], Y[kC / 8][4];
      load_vt(static_cast<const T*>(p.o.ptr) + b * p.o.sb + t0 * p.o.sl + h * p.o.sh + d0, p.o.sl, rows, cols, lane, dO);
      store_acc(p.dstates + ((head * p.n + ch) * p.dvp + d0) * DKP, DKP, lane, S);
      zero(Y);
      const uint32_t sk = smem_u32(s.k[0]), sq = smem_u32(s.q[0]);
#pragma unroll
      for (int kb = 0; kb < DKP / 16; ++kb) {
        uint32_t a[3][4];
        acc_to_a<3>(S, kb, a);
#pragma unroll
        for (int jp = 0; jp < kC / 16; ++jp)
#pragma unroll
          for (int pb = 0; pb < NP; ++pb) {
            uint32_t bf[4];
            load_b<DKP>(bf, sk + pb * (kC * DKP * 2), 2 * jp, kb, lane);
            mma_pieces<3, 2>(Y[2 * jp], Y[2 * jp + 1], a, bf, pb);
          }
      }
#pragma unroll
      for (int j = 0; j < kC / 8; ++j) {
        const float2 la = *reinterpret_cast<const float2*>(s.vec + kC + 8 * j + 2 * t);
#pragma unroll
        for (int e = 0; e < 4; ++e) Y[j][e] *= e & 1 ? la.y : la.x;
      }
      tri_product<NP, 3, 2, true>(Y, dO, smem_u32(s.pm[0]), lane);
      float X[kC / 8][4];
      zero(X);
      tri_product<3, 3, 2, true>(X, Y, smem_u32(s.t[0]), lane);
      store_acc(p.dxs + ((head * p.n + ch) * p.dvp + d0) * kC, kC, lane, X);
#pragma unroll
      for (int j = 0; j < kC / 8; ++j) {
        const float2 eg = *reinterpret_cast<const float2*>(s.vec + 8 * j + 2 * t);
        const float2 be = *reinterpret_cast<const float2*>(s.vec + 2 * kC + 8 * j + 2 * t);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          Y[j][e] = X[j][e] * (e & 1 ? be.y : be.x);
          dO[j][e] *= p.scale * (e & 1 ? eg.y : eg.x);
          X[j][e] = Y[j][e] * (e & 1 ? eg.y : eg.x);
        }
      }
      store_vt(static_cast<T*>(const_cast<void*>(p.dv.ptr)) + b * p.dv.sb + t0 * p.dv.sl + h * p.dv.sh + d0, p.dv.sl,
               rows, cols, lane, Y);
      state_add<NP, DKP>(S, s.vec[kC - 1], 1.0f, dO, sq, lane);
      state_add<NP, DKP>(S, 1.0f, -1.0f, X, sk, lane);
    }
    __syncthreads();
    if (threadIdx.x == 0 && it + kStages < p.n) chain_load(stage[st], p, b, h, p.n - 1 - it - kStages, &bar[st]);
  }
  if (cols > 0 && p.last != nullptr) state_store(p.last + head * p.dkw * p.dvw, p.dkw, p.dvw, d0, lane, S);
}

// ================================================================================================
// Backward, all chunks at once: one CTA of eight warps per (chunk, value head, batch).  With
//   E1 = dO S^T,  E2 = dX S^T,  E3 = U dS'^T,  N = -tril(D dX U^T, -1),  M = scale tril(D dO U^T, -1),
//   m_i = scale dO_i.U_i (the diagonal, where D = 1 has no gradient)
//   H = N K - e^G E2                         (the gradient of beta k)
//   dQ = scale e^G E1 + M K,   dK = beta H + C,  C = N^T (beta K) + M^T Q + e^(G_last - G) E3
//   dbeta_i = dX_i.V_i + k_i.H_i
//   dG_i = q_i.dQ_i + beta_i k_i.H_i - k_i.C_i;  the last position also gets
//          sum_i e^(G_last - G_i) k_i.E3_i + e^G_last <S, dS'>
// after which dQ_i gets m_i k_i and dK_i gets m_i q_i;
// dg is dG summed from the end of the chunk.  Every exponent's gradient is thus a row product of
// gradients that are formed anyway; k.k and q.k are not needed again.
// A warp takes 16 rows and half of the columns; dv is walked 32 channels at a time.
// ================================================================================================
constexpr int kSlab = 32;
template <int NP, int DKP>
struct alignas(128) BwdSmem {
  __nv_bfloat16 k[NP][kC * DKP], q[NP][kC * DKP];
  float vec[kVec];
  float S[kSlab][DKP + 4], dS[kSlab][DKP + 4];
  float U[kSlab][kC + 4], dX[kSlab][kC + 4];
  float dO[kC][kSlab + 8];
  float N[kC][kC + 8], M[kC][kC + 8];
  float dots[4][2][kC];         // q.dQ, k.H, k.C, e^(G_last - G) k.E3; by column half
  float dxv[4][kC];             // dX.V by quarter of the slab
  float sds[8];                 // <S, dS'> by warp
  float m[kC];                  // the diagonal of M
  uint64_t bar;
};

// A operand (16 rows from row0, k block kb) in NA pieces from a float tile stored [m][k], rows `scale`d.
template <int NA, int W>
__device__ __forceinline__ void a_rows(const float (*m)[W], int row0, int k0, int lane, uint32_t (&a)[NA][4]) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const float2 x = *reinterpret_cast<const float2*>(&m[row0 + g + 8 * (r & 1)][k0 + 2 * t + 8 * (r >> 1)]);
    uint32_t p[NA];
    split<NA>(x.x, x.y, p);
#pragma unroll
    for (int i = 0; i < NA; ++i) a[i][r] = p[i];
  }
}
// The same from a tile stored [k][m]; w (or null) scales position k.
template <int NA, int W>
__device__ __forceinline__ void a_cols(const float (*m)[W], int row0, int k0, int lane, const float* w,
                                       uint32_t (&a)[NA][4]) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int k = k0 + 2 * t + 8 * (r >> 1), i = row0 + g + 8 * (r & 1);
    float x0 = m[k][i], x1 = m[k + 1][i];
    if (w != nullptr) {
      x0 *= w[k];
      x1 *= w[k + 1];
    }
    uint32_t p[NA];
    split<NA>(x0, x1, p);
#pragma unroll
    for (int i2 = 0; i2 < NA; ++i2) a[i2][r] = p[i2];
  }
}
// B operand (k block from k0, n tile from n0) in three pieces from a float tile stored [k][n].
template <int W>
__device__ __forceinline__ void b_cols(const float (*m)[W], int k0, int n0, int lane, uint32_t (&b)[3][2]) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    uint32_t p[3];
    split<3>(m[k0 + 2 * t + 8 * r][n0 + g], m[k0 + 2 * t + 1 + 8 * r][n0 + g], p);
#pragma unroll
    for (int i = 0; i < 3; ++i) b[i][r] = p[i];
  }
}
template <int NA>
__device__ __forceinline__ void mma_all(float (&d)[4], const uint32_t (&a)[NA][4], const uint32_t (&b)[3][2]) {
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (i + j <= 2) mma_bf16(d, a[i], b[j][0], b[j][1]);
}
// d (tiles of 8 columns from col0) += a (kC positions, given by fragment loader) x tile [c][dk] in NP pieces
template <int NP, int DKP, int NT, typename F>
__device__ __forceinline__ void add_rows_times_tile(float (&d)[NT][4], uint32_t tile, int col_tile0, int kb0, int kb1,
                                                    int lane, F frag) {
  for (int kb = kb0; kb < kb1; ++kb) {
    uint32_t a[3][4];
    frag(kb, a);
#pragma unroll
    for (int jp = 0; jp < NT / 2; ++jp)
#pragma unroll
      for (int pb = 0; pb < NP; ++pb) {
        uint32_t bf[4];
        load_bt<DKP>(bf, tile + pb * (kC * DKP * 2), col_tile0 + 2 * jp, kb, lane);
        mma_pieces<3, 2>(d[2 * jp], d[2 * jp + 1], a, bf, pb);
      }
  }
}

template <typename T, int NP, int DKP>
__global__ void __launch_bounds__(256) delta_bwd_chunk(const __grid_constant__ DeltaParams p) {
  extern __shared__ __align__(128) unsigned char smem_raw[];
  auto& s = *reinterpret_cast<BwdSmem<NP, DKP>*>(smem_raw);
  constexpr int NT = DKP / 16;                    // n tiles of a warp's half of dk
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int row0 = 16 * (warp & 3), half = warp >> 2;
  const int ch = blockIdx.x, h = blockIdx.y, b = blockIdx.z, hk = h / p.group;
  const int rows = min(kC, p.L - ch * kC);
  const long long t0 = (long long)ch * kC;
  const size_t at = ((size_t)b * p.Hv + h) * p.n + ch;
  const size_t atk = ((size_t)b * p.Hk + hk) * p.n + ch;
  if (tid == 0) {
    mbar_init(&s.bar, 1);
    fence_mbar_init();
    mbar_arrive_expect_tx(&s.bar, sizeof(s.k) + sizeof(s.q) + sizeof(s.vec));
    bulk_load(s.k, p.kimg + atk * (NP * kC * DKP), sizeof(s.k), &s.bar);
    bulk_load(s.q, p.qimg + atk * (NP * kC * DKP), sizeof(s.q), &s.bar);
    bulk_load(s.vec, p.vec + at * kVec, sizeof(s.vec), &s.bar);
  }
  float E1[NT][4], E2[NT][4], E3[NT][4], XU[4][4], OU[4][4];
  zero(E1);
  zero(E2);
  zero(E3);
  zero(XU);
  zero(OU);
  float dot = 0.0f, dxv = 0.0f;
  const T* dOb = static_cast<const T*>(p.o.ptr) + b * p.o.sb + t0 * p.o.sl + h * p.o.sh;
  const T* Vb = static_cast<const T*>(p.v.ptr) + b * p.v.sb + t0 * p.v.sl + h * p.v.sh;
  for (int v0 = 0; v0 < p.dvp; v0 += kSlab) {
    const int vn = min(kSlab, p.dvp - v0);
    __syncthreads();
    for (int e = tid; e < kSlab * DKP / 4; e += 256) {
      const int r = e / (DKP / 4), c = 4 * (e % (DKP / 4));
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
      if (r < vn) {
        x = *reinterpret_cast<const float4*>(p.states + (at * p.dvp + v0 + r) * DKP + c);
        y = *reinterpret_cast<const float4*>(p.dstates + (at * p.dvp + v0 + r) * DKP + c);
      }
      *reinterpret_cast<float4*>(&s.S[r][c]) = x;
      *reinterpret_cast<float4*>(&s.dS[r][c]) = y;
      dot = fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, fmaf(x.w, y.w, dot))));
    }
    for (int e = tid; e < kSlab * kC / 4; e += 256) {
      const int r = e / (kC / 4), c = 4 * (e % (kC / 4));
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
      if (r < vn) {
        x = *reinterpret_cast<const float4*>(p.us + (at * p.dvp + v0 + r) * kC + c);
        y = *reinterpret_cast<const float4*>(p.dxs + (at * p.dvp + v0 + r) * kC + c);
      }
      *reinterpret_cast<float4*>(&s.U[r][c]) = x;
      *reinterpret_cast<float4*>(&s.dX[r][c]) = y;
    }
    for (int e = tid; e < kC * kSlab; e += 256) {
      const int c = e / kSlab, d = e % kSlab;
      s.dO[c][d] = c < rows && v0 + d < p.dvw ? to_f32(dOb[c * p.o.sl + v0 + d]) : 0.0f;
    }
    __syncthreads();
    {
      const int c = tid & 63, d1 = (tid >> 6) * 8;
      if (c < rows)
#pragma unroll
        for (int d = d1; d < d1 + 8; ++d)
          if (v0 + d < p.dvw) dxv = fmaf(s.dX[d][c], to_f32(Vb[c * p.v.sl + v0 + d]), dxv);
    }
#pragma unroll
    for (int k0 = 0; k0 < kSlab; k0 += 16) {
      uint32_t ao[NP][4], ax[3][4], au[3][4];
      a_rows<NP>(s.dO, row0, k0, lane, ao);
      a_cols<3>(s.dX, row0, k0, lane, nullptr, ax);
      a_cols<3>(s.U, row0, k0, lane, nullptr, au);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        uint32_t bf[3][2];
        b_cols(s.S, k0, half * (DKP / 2) + 8 * j, lane, bf);
        mma_all<NP>(E1[j], ao, bf);
        mma_all<3>(E2[j], ax, bf);
        b_cols(s.dS, k0, half * (DKP / 2) + 8 * j, lane, bf);
        mma_all<3>(E3[j], au, bf);
      }
      if (row0 + 15 >= 32 * half) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t bf[3][2];
          b_cols(s.U, k0, 32 * half + 8 * j, lane, bf);
          mma_all<3>(XU[j], ax, bf);
          mma_all<NP>(OU[j], ao, bf);
        }
      }
    }
  }
  mbar_wait(&s.bar, 0, p.err);
  // N and M
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = row0 + g + 8 * (e >> 1), c = 32 * half + 8 * j + 2 * t + (e & 1);
      const float d = i >= c ? ex2((s.vec[3 * kC + i] - s.vec[3 * kC + c]) + (s.vec[4 * kC + i] - s.vec[4 * kC + c])) : 0.0f;
      s.N[i][c] = i > c ? -d * XU[j][e] : 0.0f;
      s.M[i][c] = i > c ? p.scale * d * OU[j][e] : 0.0f;
      if (i == c) s.m[i] = p.scale * OU[j][e];
    }
  s.dxv[tid >> 6][tid & 63] = dxv;
  dot = group_allreduce<32, 1>(dot);
  if (lane == 0) s.sds[warp] = dot;
  __syncthreads();
  const uint32_t sk = smem_u32(s.k[0]), sq = smem_u32(s.q[0]);
  const int ct = half * NT;
  const float* beta = s.vec + 2 * kC;
  float eg[2], la[2], be[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    eg[r] = s.vec[row0 + g + 8 * r];
    la[r] = s.vec[kC + row0 + g + 8 * r];
    be[r] = beta[row0 + g + 8 * r];
  }
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      E1[j][e] *= p.scale * eg[e >> 1];
      E2[j][e] *= -eg[e >> 1];
      E3[j][e] *= la[e >> 1];
    }
  // x.y of the warp's rows over its columns, from a tile in pieces
  auto row_dot = [&](const float (&c)[NT][4], const __nv_bfloat16* tile, float (&out)[2]) {
    out[0] = out[1] = 0.0f;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int off = tile_off<DKP>(row0 + g + 8 * r, ct + j) + 2 * t;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const uint32_t w = *reinterpret_cast<const uint32_t*>(tile + i * (kC * DKP) + off);
          out[r] = fmaf(lo_f32(w), c[j][2 * r], fmaf(hi_f32(w), c[j][2 * r + 1], out[r]));
        }
      }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      out[r] += __shfl_xor_sync(0xffffffffu, out[r], 1);
      out[r] += __shfl_xor_sync(0xffffffffu, out[r], 2);
    }
  };
  auto put_dot = [&](int which, const float (&c)[NT][4], const __nv_bfloat16* tile) {
    float d[2];
    row_dot(c, tile, d);
    if (t == 0) {
      s.dots[which][half][row0 + g] = d[0];
      s.dots[which][half][row0 + g + 8] = d[1];
    }
  };
  const int w4 = warp & 3;
  put_dot(3, E3, s.k[0]);
  // dQ = scale e^G E1 + M K
  add_rows_times_tile<NP, DKP>(E1, sk, ct, 0, w4 + 1, lane,
                               [&](int kb, uint32_t (&a)[3][4]) { a_rows<3>(s.M, row0, 16 * kb, lane, a); });
  put_dot(0, E1, s.q[0]);
  // H = N K - e^G E2
  add_rows_times_tile<NP, DKP>(E2, sk, ct, 0, w4 + 1, lane,
                               [&](int kb, uint32_t (&a)[3][4]) { a_rows<3>(s.N, row0, 16 * kb, lane, a); });
  put_dot(1, E2, s.k[0]);
  // C = N^T (beta K) + M^T Q + e^(G_last - G) E3
  add_rows_times_tile<NP, DKP>(E3, sk, ct, w4, kC / 16, lane,
                               [&](int kb, uint32_t (&a)[3][4]) { a_cols<3>(s.N, row0, 16 * kb, lane, beta, a); });
  add_rows_times_tile<NP, DKP>(E3, sq, ct, w4, kC / 16, lane,
                               [&](int kb, uint32_t (&a)[3][4]) { a_cols<3>(s.M, row0, 16 * kb, lane, nullptr, a); });
  put_dot(2, E3, s.k[0]);
  // query and key gradients: to the tensors, or per value head where key heads are shared
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = row0 + g + 8 * (e >> 1), c = 8 * (ct + j) + 2 * t + (e & 1);
      if (i >= rows || c >= p.dkw) continue;
      float kv = 0.0f, qv = 0.0f;
#pragma unroll
      for (int x = 0; x < NP; ++x) {
        const int off = x * (kC * DKP) + tile_off<DKP>(i, ct + j) + 2 * t + (e & 1);
        kv += __bfloat162float(s.k[0][off]);
        qv += __bfloat162float(s.q[0][off]);
      }
      const float dq = fmaf(s.m[i], kv, E1[j][e]);
      const float dk = fmaf(s.m[i], qv, fmaf(be[e >> 1], E2[j][e], E3[j][e]));
      if (p.group > 1) {
        const size_t o = (((size_t)b * p.L + t0 + i) * p.Hv + h) * p.dkw + c;
        p.pdq[o] = dq;
        p.pdk[o] = dk;
      } else {
        static_cast<T*>(const_cast<void*>(p.dq.ptr))[b * p.dq.sb + (t0 + i) * p.dq.sl + hk * p.dq.sh + c] = from_f32<T>(dq);
        static_cast<T*>(const_cast<void*>(p.dk.ptr))[b * p.dk.sb + (t0 + i) * p.dk.sl + hk * p.dk.sh + c] = from_f32<T>(dk);
      }
    }
  __syncthreads();
  if (warp == 0) {
    float dG[2], tail = 0.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = 2 * lane + i;
      const float kH = s.dots[1][0][r] + s.dots[1][1][r];
      dG[i] = (s.dots[0][0][r] + s.dots[0][1][r]) + beta[r] * kH - (s.dots[2][0][r] + s.dots[2][1][r]);
      tail += s.dots[3][0][r] + s.dots[3][1][r];
      if (r < rows)
        p.dbeta[((size_t)b * p.L + t0 + r) * p.Hv + h] =
            ((s.dxv[0][r] + s.dxv[1][r]) + (s.dxv[2][r] + s.dxv[3][r])) + kH;
    }
    tail = group_allreduce<32, 1>(tail);
    float sds = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sds += s.sds[i];
    tail = fmaf(s.vec[kC - 1], sds, tail);
    float run = dG[0] + dG[1];
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const float down = __shfl_down_sync(0xffffffffu, run, m);
      if (lane + m < 32) run += down;
    }
    run += tail;
    if (2 * lane < rows) p.dg[((size_t)b * p.L + t0 + 2 * lane) * p.Hv + h] = run;
    if (2 * lane + 1 < rows) p.dg[((size_t)b * p.L + t0 + 2 * lane + 1) * p.Hv + h] = run - dG[0];
  }
}

// dq, dk (B, L, Hk, dk): the value heads' parts summed in head order.
template <typename T>
__global__ void __launch_bounds__(256) delta_sum_heads(const __grid_constant__ DeltaParams p) {
  const long long i = blockIdx.x * 256LL + threadIdx.x;
  const long long total = (long long)p.B * p.L * p.Hk * p.dkw;
  if (i >= total) return;
  const int c = (int)(i % p.dkw), hk = (int)(i / p.dkw % p.Hk);
  const long long row = i / p.dkw / p.Hk, b = row / p.L, l = row % p.L;
  float dq = 0.0f, dk = 0.0f;
  for (int r = 0; r < p.group; ++r) {
    const size_t o = ((size_t)row * p.Hv + hk * p.group + r) * p.dkw + c;
    dq += p.pdq[o];
    dk += p.pdk[o];
  }
  static_cast<T*>(const_cast<void*>(p.dq.ptr))[b * p.dq.sb + l * p.dq.sl + hk * p.dq.sh + c] = from_f32<T>(dq);
  static_cast<T*>(const_cast<void*>(p.dk.ptr))[b * p.dk.sb + l * p.dk.sl + hk * p.dk.sh + c] = from_f32<T>(dk);
}

// ================================================================================================
// One token: S <- a S, e = beta (v - S^T k), S <- S + k e^T, o = scale S^T q.
// A CTA of 256 threads takes 32 value channels (lanes) of one head; its warps share the dk rows.  Two
// passes over rows held in registers: the state is read and written once, which bounds the kernel.
// ================================================================================================
constexpr int kStepRows = 16;                     // dk rows per warp: 8 warps cover dk <= 128
template <typename T>
__global__ void __launch_bounds__(256) delta_step(const __grid_constant__ DeltaParams p) {
  __shared__ float red[2][8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h = blockIdx.y, b = blockIdx.z, hk = h / p.group;
  const int d = blockIdx.x * 32 + lane;
  const bool live = d < p.dvw;
  float* S = p.last + ((size_t)b * p.Hv + h) * p.dkw * p.dvw + d;
  const T* kp = static_cast<const T*>(p.k.ptr) + b * p.k.sb + hk * p.k.sh;
  const T* qp = static_cast<const T*>(p.q.ptr) + b * p.q.sb + hk * p.q.sh;
  float x[kStepRows], kr[kStepRows], part = 0.0f;
  const float alpha = expf(p.g[b * p.gsb + h]), beta = p.beta[b * p.bsb + h];
#pragma unroll
  for (int i = 0; i < kStepRows; ++i) {
    const int r = warp + 8 * i;
    x[i] = live && r < p.dkw ? S[(size_t)r * p.dvw] : 0.0f;
    kr[i] = r < p.dkw ? to_f32(kp[r]) : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < kStepRows; ++i) {
    x[i] *= alpha;
    part = fmaf(x[i], kr[i], part);
  }
  red[0][warp][lane] = part;
  __syncthreads();
  float dot = 0.0f;
#pragma unroll
  for (int w = 0; w < 8; ++w) dot += red[0][w][lane];
  const float v = live ? to_f32(static_cast<const T*>(p.v.ptr)[b * p.v.sb + h * p.v.sh + d]) : 0.0f;
  const float e = beta * (v - dot);
  part = 0.0f;
#pragma unroll
  for (int i = 0; i < kStepRows; ++i) {
    const int r = warp + 8 * i;
    x[i] = fmaf(kr[i], e, x[i]);
    if (r < p.dkw) {
      part = fmaf(x[i], to_f32(qp[r]), part);
      if (live) S[(size_t)r * p.dvw] = x[i];
    }
  }
  red[1][warp][lane] = part;
  __syncthreads();
  if (warp == 0 && live) {
    float o = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) o += red[1][w][lane];
    static_cast<T*>(const_cast<void*>(p.o.ptr))[b * p.o.sb + h * p.o.sh + d] = from_f32<T>(p.scale * o);
  }
}

// ================================================================================================
// Host
// ================================================================================================
template <typename... A>
int fail(int code, const char* fmt, A... a) {
  if constexpr (sizeof...(A) == 0) {
    return report_error(code, fmt);
  } else {
    char msg[256];
    snprintf(msg, sizeof(msg), fmt, a...);
    return report_error(code, msg);
  }
}

Heads heads(const ssm_heads& v) { return Heads{v.ptr, v.batch_stride, v.row_stride, v.head_stride}; }

struct Shape {
  int64_t B, L, Hk, Hv, dk, dv;
  int dtype;
  int np() const { return dtype == SSM_BF16 ? 1 : 3; }
  int dkp() const { return dk <= 64 ? 64 : 128; }
  int64_t dvp() const { return (dv + 15) / 16 * 16; }
  int64_t n() const { return (L + kC - 1) / kC; }
};

int check_shape(const Shape& s) {
  if (s.B < 1 || s.L < 1 || s.Hk < 1 || s.Hv < 1 || s.dk < 1 || s.dv < 1)
    return fail(SSM_ERR_INVALID, "gated delta rule: batch, length, heads and widths must be positive");
  if (s.Hv % s.Hk != 0)
    return fail(SSM_ERR_INVALID, "gated delta rule: %lld value heads are not a multiple of %lld key heads",
                (long long)s.Hv, (long long)s.Hk);
  if (s.dk > 128) return fail(SSM_ERR_UNSUPPORTED, "gated delta rule: key width %lld above 128", (long long)s.dk);
  if (s.B > 65535 || s.Hv > 65535 || s.dv > (1 << 20) || s.L > (1LL << 30))
    return fail(SSM_ERR_INVALID, "gated delta rule: shape out of range (B=%lld, L=%lld)", (long long)s.B, (long long)s.L);
  if (s.dtype != SSM_F32 && s.dtype != SSM_BF16) return fail(SSM_ERR_DTYPE, "gated delta rule: dtype %d unsupported", s.dtype);
  return SSM_OK;
}
int check_heads(const char* name, const ssm_heads& v, int dtype) {
  if (v.ptr == nullptr) return fail(SSM_ERR_INVALID, "gated delta rule: %s is required", name);
  if (v.dtype != dtype) return fail(SSM_ERR_DTYPE, "gated delta rule: %s must have q's dtype", name);
  return SSM_OK;
}
int check_gate(const char* name, const ssm_view& v) {
  if (v.ptr == nullptr) return fail(SSM_ERR_INVALID, "gated delta rule: %s is required", name);
  if (v.dtype != SSM_F32) return fail(SSM_ERR_DTYPE, "gated delta rule: %s must be float32", name);
  return SSM_OK;
}

struct Carver {
  unsigned char* base;
  size_t used = 0;
  template <typename T>
  T* take(size_t count) {
    T* r = reinterpret_cast<T*>(base + used);
    used += (count * sizeof(T) + 255) & ~size_t(255);
    return r;
  }
};

// The workspace's parts; with base null only its size is of use.
size_t carve(const Shape& s, bool bwd, DeltaParams& p, unsigned char* base) {
  Carver c{base};
  const size_t chunks_k = (size_t)s.B * s.Hk * s.n(), chunks = (size_t)s.B * s.Hv * s.n();
  p.kimg = c.take<__nv_bfloat16>(chunks_k * s.np() * kC * s.dkp());
  p.qimg = c.take<__nv_bfloat16>(chunks_k * s.np() * kC * s.dkp());
  p.timg = c.take<__nv_bfloat16>(chunks * 3 * kTri);
  p.pimg = c.take<__nv_bfloat16>(chunks * 3 * kTri);
  p.vec = c.take<float>(chunks * kVec);
  if (bwd) {
    p.dstates = c.take<float>(chunks * s.dvp() * s.dkp());
    p.dxs = c.take<float>(chunks * s.dvp() * kC);
    if (s.Hv > s.Hk) {
      p.pdq = c.take<float>((size_t)s.B * s.L * s.Hv * s.dk);
      p.pdk = c.take<float>((size_t)s.B * s.L * s.Hv * s.dk);
    }
  }
  return c.used + 256;
}
unsigned char* align256(void* p) {
  return reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(p) + 255) & ~uintptr_t(255));
}

void fill(DeltaParams& p, const Shape& s, ssm_heads q, ssm_heads k, ssm_heads v, ssm_view g, ssm_view beta, float scale) {
  p.q = heads(q);
  p.k = heads(k);
  p.v = heads(v);
  p.g = static_cast<const float*>(g.ptr);
  p.gsb = g.batch_stride;
  p.gsl = g.row_stride;
  p.beta = static_cast<const float*>(beta.ptr);
  p.bsb = beta.batch_stride;
  p.bsl = beta.row_stride;
  p.B = (int)s.B;
  p.L = (int)s.L;
  p.Hk = (int)s.Hk;
  p.Hv = (int)s.Hv;
  p.dkw = (int)s.dk;
  p.dvw = (int)s.dv;
  p.dvp = (int)s.dvp();
  p.n = (int)s.n();
  p.group = (int)(s.Hv / s.Hk);
  p.scale = scale;
  p.err = device_error_word();
}

template <typename K>
cudaError_t launch(K kern, dim3 grid, int threads, size_t smem, const DeltaParams& p, cudaStream_t st) {
  if (smem > 48 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  kern<<<grid, threads, smem, st>>>(p);
  return cudaGetLastError();
}

// Warps per CTA of the chain kernels, 16 value channels each: up to eight, four where eight would leave
// SMs without a CTA (a warp then has a scheduler to itself either way).
int chain_warps(const Shape& s) {
  const int64_t tiles = s.dvp() / 16;
  int w = 1;
  while (w < 8 && w < tiles) w *= 2;
  return w == 8 && s.B * s.Hv * ((tiles + 7) / 8) < 148 ? 4 : w;
}

template <typename T, int NP, int DKP>
cudaError_t run_fwd(const Shape& s, const DeltaParams& p, cudaStream_t st) {
  const dim3 grid((unsigned)s.n(), (unsigned)s.Hv, (unsigned)s.B);
  cudaError_t e = launch(delta_prep<T, NP, DKP>, grid, 128, sizeof(PrepSmem<T, NP, DKP>), p, st);
  if (e != cudaSuccess) return e;
  constexpr int PP = NP == 1 ? 2 : 3;
  const int w = chain_warps(s);
  const dim3 cg((unsigned)((s.dvp() / 16 + w - 1) / w), (unsigned)s.Hv, (unsigned)s.B);
  constexpr size_t smem = chain_smem<NP, DKP, PP>();
  return p.states != nullptr ? launch(delta_fwd<T, NP, DKP, true>, cg, 32 * w, smem, p, st)
                             : launch(delta_fwd<T, NP, DKP, false>, cg, 32 * w, smem, p, st);
}

template <typename T, int NP, int DKP>
cudaError_t run_bwd(const Shape& s, const DeltaParams& p, cudaStream_t st) {
  const dim3 grid((unsigned)s.n(), (unsigned)s.Hv, (unsigned)s.B);
  cudaError_t e = launch(delta_prep<T, NP, DKP>, grid, 128, sizeof(PrepSmem<T, NP, DKP>), p, st);
  if (e != cudaSuccess) return e;
  const int w = chain_warps(s);
  const dim3 cg((unsigned)((s.dvp() / 16 + w - 1) / w), (unsigned)s.Hv, (unsigned)s.B);
  e = launch(delta_bwd_chain<T, NP, DKP>, cg, 32 * w, chain_smem<NP, DKP, 3>(), p, st);
  if (e != cudaSuccess) return e;
  e = launch(delta_bwd_chunk<T, NP, DKP>, grid, 256, sizeof(BwdSmem<NP, DKP>), p, st);
  if (e != cudaSuccess || p.group == 1) return e;
  const long long total = (long long)p.B * p.L * p.Hk * p.dkw;
  return launch(delta_sum_heads<T>, dim3((unsigned)((total + 255) / 256)), 256, 0, p, st);
}

}  // namespace

extern "C" {

int ssm_gated_delta_workspace_size(int64_t B, int64_t L, int64_t Hk, int64_t Hv, int64_t dk, int64_t dv, int32_t dtype,
                                   int32_t backward, size_t* bytes) {
  if (bytes == nullptr) return fail(SSM_ERR_INVALID, "gated delta rule: bytes is NULL");
  const Shape s{B, L, Hk, Hv, dk, dv, dtype};
  int rc = check_shape(s);
  if (rc) return rc;
  DeltaParams p;
  *bytes = carve(s, backward != 0, p, nullptr);
  return SSM_OK;
}

int ssm_gated_delta_saved_size(int64_t B, int64_t L, int64_t Hk, int64_t Hv, int64_t dk, int64_t dv, int32_t dtype,
                               size_t* bytes) {
  if (bytes == nullptr) return fail(SSM_ERR_INVALID, "gated delta rule: bytes is NULL");
  const Shape s{B, L, Hk, Hv, dk, dv, dtype};
  int rc = check_shape(s);
  if (rc) return rc;
  *bytes = (size_t)B * Hv * s.n() * s.dvp() * (s.dkp() + kC) * sizeof(float) + 256;
  return SSM_OK;
}

static void saved_parts(const Shape& s, void* saved, DeltaParams& p) {
  p.states = reinterpret_cast<float*>(align256(saved));
  p.us = p.states + (size_t)s.B * s.Hv * s.n() * s.dvp() * s.dkp();
}

int ssm_gated_delta_fwd(int64_t B, int64_t L, int64_t Hk, int64_t Hv, int64_t dk, int64_t dv, ssm_heads q, ssm_heads k,
                        ssm_heads v, ssm_view g, ssm_view beta, const float* h0, float scale, ssm_heads o, float* last,
                        void* saved, void* workspace, size_t workspace_bytes, void* stream) {
  const Shape s{B, L, Hk, Hv, dk, dv, q.dtype};
  int rc = check_shape(s);
  if (rc) return rc;
  if ((rc = check_heads("q", q, s.dtype)) || (rc = check_heads("k", k, s.dtype)) || (rc = check_heads("v", v, s.dtype)) ||
      (rc = check_heads("o", o, s.dtype)) || (rc = check_gate("g", g)) || (rc = check_gate("beta", beta)))
    return rc;
  DeltaParams p;
  memset(&p, 0, sizeof(p));
  const size_t need = carve(s, false, p, nullptr);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(SSM_ERR_WORKSPACE, "gated delta rule: forward workspace of %zu bytes required, %zu given", need,
                workspace_bytes);
  carve(s, false, p, align256(workspace));
  fill(p, s, q, k, v, g, beta, scale);
  p.o = heads(o);
  p.h0 = h0;
  p.last = last;
  if (saved != nullptr) saved_parts(s, saved, p);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (s.dtype == SSM_BF16)
    e = s.dkp() == 64 ? run_fwd<__nv_bfloat16, 1, 64>(s, p, st) : run_fwd<__nv_bfloat16, 1, 128>(s, p, st);
  else
    e = s.dkp() == 64 ? run_fwd<float, 3, 64>(s, p, st) : run_fwd<float, 3, 128>(s, p, st);
  if (e != cudaSuccess) return fail(SSM_ERR_CUDA, "gated delta rule forward: %s", cudaGetErrorString(e));
  return SSM_OK;
}

int ssm_gated_delta_bwd(int64_t B, int64_t L, int64_t Hk, int64_t Hv, int64_t dk, int64_t dv, ssm_heads q, ssm_heads k,
                        ssm_heads v, ssm_view g, ssm_view beta, float scale, const void* saved, ssm_heads d_o,
                        const float* dlast, ssm_heads d_q, ssm_heads d_k, ssm_heads d_v, float* d_g, float* d_beta,
                        float* dh0, void* workspace, size_t workspace_bytes, void* stream) {
  const Shape s{B, L, Hk, Hv, dk, dv, q.dtype};
  int rc = check_shape(s);
  if (rc) return rc;
  if ((rc = check_heads("q", q, s.dtype)) || (rc = check_heads("k", k, s.dtype)) || (rc = check_heads("v", v, s.dtype)) ||
      (rc = check_heads("do", d_o, s.dtype)) || (rc = check_heads("dq", d_q, s.dtype)) ||
      (rc = check_heads("dk", d_k, s.dtype)) || (rc = check_heads("dv", d_v, s.dtype)) || (rc = check_gate("g", g)) ||
      (rc = check_gate("beta", beta)))
    return rc;
  if (saved == nullptr || d_g == nullptr || d_beta == nullptr)
    return fail(SSM_ERR_INVALID, "gated delta rule: saved, dg and dbeta are required");
  DeltaParams p;
  memset(&p, 0, sizeof(p));
  const size_t need = carve(s, true, p, nullptr);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(SSM_ERR_WORKSPACE, "gated delta rule: backward workspace of %zu bytes required, %zu given", need,
                workspace_bytes);
  carve(s, true, p, align256(workspace));
  fill(p, s, q, k, v, g, beta, scale);
  saved_parts(s, const_cast<void*>(saved), p);
  p.o = heads(d_o);
  p.dq = heads(d_q);
  p.dk = heads(d_k);
  p.dv = heads(d_v);
  p.dg = d_g;
  p.dbeta = d_beta;
  p.h0 = dlast;
  p.last = dh0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (s.dtype == SSM_BF16)
    e = s.dkp() == 64 ? run_bwd<__nv_bfloat16, 1, 64>(s, p, st) : run_bwd<__nv_bfloat16, 1, 128>(s, p, st);
  else
    e = s.dkp() == 64 ? run_bwd<float, 3, 64>(s, p, st) : run_bwd<float, 3, 128>(s, p, st);
  if (e != cudaSuccess) return fail(SSM_ERR_CUDA, "gated delta rule backward: %s", cudaGetErrorString(e));
  return SSM_OK;
}

int ssm_gated_delta_state_update(int64_t B, int64_t Hk, int64_t Hv, int64_t dk, int64_t dv, float* state, ssm_heads q,
                                 ssm_heads k, ssm_heads v, ssm_view g, ssm_view beta, float scale, ssm_heads o,
                                 void* stream) {
  const Shape s{B, 1, Hk, Hv, dk, dv, q.dtype};
  int rc = check_shape(s);
  if (rc) return rc;
  if ((rc = check_heads("q", q, s.dtype)) || (rc = check_heads("k", k, s.dtype)) || (rc = check_heads("v", v, s.dtype)) ||
      (rc = check_heads("o", o, s.dtype)) || (rc = check_gate("g", g)) || (rc = check_gate("beta", beta)))
    return rc;
  if (state == nullptr) return fail(SSM_ERR_INVALID, "gated delta rule: state is required");
  DeltaParams p;
  memset(&p, 0, sizeof(p));
  fill(p, s, q, k, v, g, beta, scale);
  p.o = heads(o);
  p.last = state;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)((dv + 31) / 32), (unsigned)Hv, (unsigned)B);
  const cudaError_t e = s.dtype == SSM_BF16 ? launch(delta_step<__nv_bfloat16>, grid, 256, 0, p, st)
                                            : launch(delta_step<float>, grid, 256, 0, p, st);
  if (e != cudaSuccess) return fail(SSM_ERR_CUDA, "gated delta state update: %s", cudaGetErrorString(e));
  return SSM_OK;
}

}  // extern "C"
