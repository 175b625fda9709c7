// ssm_delta.cu — the gated delta rule: chunked forward and backward, one-token state update.
// The formulas are in ssm_delta.cuh.  Forward: delta_prep (everything that does not need the state, all
// chunks at once), delta_fwd (the state from chunk to chunk, and the output).  Backward: delta_bwd_chain (the
// state's gradient from the last chunk to the first), delta_bwd_chunk (all other gradients, all chunks at
// once), delta_sum_heads (query and key gradients over the value heads that share a key head).
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdio>
#include <cstring>

#include "ssm_b200.h"
#include "ssm_delta.cuh"
#include "ssm_delta_chunk.cuh"
#include "ssm_delta_tc.cuh"
#include "ssm_launch.cuh"

namespace ssm {
int report_error(int code, const char* msg);
int* device_error_word();
}  // namespace ssm

namespace {

using namespace ssm;

constexpr int kPitch = kC + 4;

// ================================================================================================
// Chunk preparation: one CTA of four warps per (chunk, value head, batch).  Short dependent steps (sums of g, two
// products, a triangular inverse) bound it, so CTAs are small, 33 KB of shared memory in bf16, five to an SM.
// 5120 chunks of 64 x 128 (bf16): 135 us; in 90 KB, with rows loaded through registers: 252 us.
// ================================================================================================
template <int NP, int DKP>
struct alignas(128) PrepSmem {
  union {
    struct {
      __nv_bfloat16 k[NP][kC * DKP], q[NP][kC * DKP];
    };
    struct {                            // after the products: A, and T in its place
      float T_[kC][kPitch], tmp[32][36];
    };
  };
  float gh[kC], gl[kC], beta[kC];
};

template <typename T, int NP, int DKP>
__global__ void __launch_bounds__(128, NP == 1 ? 5 : 2) delta_prep(const __grid_constant__ DeltaParams p) {
  extern __shared__ __align__(128) unsigned char smem_raw[];
  auto& s = *reinterpret_cast<PrepSmem<NP, DKP>*>(smem_raw);
  const int ch = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int t0 = ch * kC, rows = min(kC, p.L - t0), hk = h / p.group;
  const size_t at = ((size_t)b * p.Hv + h) * p.n + ch;
  const size_t atk = ((size_t)b * p.Hk + hk) * p.n + ch;

  // q and k in pieces: into shared memory and, once per key head, into the tiles the other kernels load
  const bool writer = h % p.group == 0;
  const T* kbase = static_cast<const T*>(p.k.ptr) + b * p.k.sb + t0 * p.k.sl + hk * p.k.sh;
  const T* qbase = static_cast<const T*>(p.q.ptr) + b * p.q.sb + t0 * p.q.sl + hk * p.q.sh;
  const bool kv = rows_aligned16(p.k, sizeof(T)), qv = rows_aligned16(p.q, sizeof(T));
  __nv_bfloat16* kg = p.kimg + atk * (NP * kC * DKP);
  __nv_bfloat16* qg = p.qimg + atk * (NP * kC * DKP);
  constexpr int kGroups = kC * DKP / 8 / 128;            // 8-element groups per thread and tensor
  const bool direct = NP == 1 && kv && qv && p.dkw % 8 == 0;   // bf16 rows are the tile's rows as they are
  if (direct) {
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      const int e = tid + 128 * i, r = e / (DKP / 8), grp = e % (DKP / 8), off = tile_off<DKP>(r, grp);
      if (r < rows && grp * 8 < p.dkw) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(&s.k[0][off])), "l"(kbase + r * p.k.sl + grp * 8) : "memory");
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(&s.q[0][off])), "l"(qbase + r * p.q.sl + grp * 8) : "memory");
      } else {
        *reinterpret_cast<uint4*>(&s.k[0][off]) = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(&s.q[0][off]) = make_uint4(0, 0, 0, 0);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  } else {
    constexpr int kBatch = 4;                              // loads in flight before the first is used
#pragma unroll 1
    for (int i0 = 0; i0 < kGroups; i0 += kBatch) {
      float x[kBatch][8], y[kBatch][8];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int e = tid + 128 * (i0 + i), r = e / (DKP / 8), grp = e % (DKP / 8), width = r < rows ? p.dkw : 0;
        load8<T>(kbase + r * p.k.sl, grp * 8, width, kv, x[i]);
        load8<T>(qbase + r * p.q.sl, grp * 8, width, qv, y[i]);
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int e = tid + 128 * (i0 + i), off = tile_off<DKP>(e / (DKP / 8), e % (DKP / 8));
        put_pieces<NP>(x[i], s.k[0], writer ? kg : nullptr, off, kC * DKP);
        put_pieces<NP>(y[i], s.q[0], writer ? qg : nullptr, off, kC * DKP);
      }
    }
  }
  // running sums of g.  In double and kept as two floats: differences of neighbours stay exact to fp32
  // also behind a position that resets the state.  exp(-1000) is 0, so -inf can be taken as -1000.
  if (warp == 0) {
    double acc[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = 2 * lane + i;
      float gate = r < rows ? p.g[b * p.gsb + (t0 + r) * p.gsl + h] : 0.0f;
      gate = gate < -1000.0f ? -1000.0f : gate;
      acc[i] = (double)gate * 1.4426950408889634;
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
    const double before = __shfl_up_sync(0xffffffffu, run, 1);
    const double G[2] = {lane > 0 ? before + acc[0] : acc[0], run};      // of its own position and those before, also where one is NaN
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
  if (direct) asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  if (direct && writer) {
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      const int e = tid + 128 * i;
      reinterpret_cast<uint4*>(kg)[e] = reinterpret_cast<const uint4*>(s.k[0])[e];
      reinterpret_cast<uint4*>(qg)[e] = reinterpret_cast<const uint4*>(s.q[0])[e];
    }
  }

  // k.k and q.k of the warp's 16 rows against the columns up to its own
  float kk[kC / 8][4];
  {
    float qk[kC / 8][4];
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
          uint32_t bf[1][4];
          load_b<DKP>(bf[0], sk + pb * (kC * DKP * 2), 2 * jp, kb, lane);
          mma_pieces<0, 2>(kk, 2 * jp, ak, bf, pb);
          mma_pieces<0, 2>(qk, 2 * jp, aq, bf, pb);
        }
      }
    }
    // P goes out as it is; A stays in registers until every warp is past the tiles that it replaces
#pragma unroll
    for (int j = 0; j < kC / 8; ++j)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int i = 16 * warp + g + 8 * r, c = 8 * j + 2 * t;
        float x[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float d = i >= c + e ? ex2((s.gh[i] - s.gh[c + e]) + (s.gl[i] - s.gl[c + e])) : 0.0f;
          x[e] = i >= c + e ? p.scale * (d * qk[j][2 * r + e]) : 0.0f;
          kk[j][2 * r + e] = i > c + e ? s.beta[i] * (d * kk[j][2 * r + e]) : 0.0f;
        }
        uint32_t q[3];
        split<3>(x[0], x[1], q);
        __nv_bfloat16* o = p.pimg + at * (3 * kTri) + tile_off<kC>(i, j) + 2 * t;
#pragma unroll
        for (int k = 0; k < 3; ++k) *reinterpret_cast<uint32_t*>(o + k * kTri) = q[k];
      }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kC / 8; ++j)
#pragma unroll
    for (int r = 0; r < 2; ++r)
      *reinterpret_cast<float2*>(&s.T_[16 * warp + g + 8 * r][8 * j + 2 * t]) = make_float2(kk[j][2 * r], kk[j][2 * r + 1]);
  __syncthreads();

  // T = (I + A)^-1 in A's place by forward substitution: the diagonal 16 x 16 blocks, then the blocks below
  // them from the blocks beside: T21 = -T22 A21 T11.
  {
    const int r0 = 16 * warp, col = lane & 15;
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v[4] = {i == col ? 1.0f : 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int m0 = 0; m0 < i; m0 += 4) {
        float a[4];
        load4(&s.T_[r0 + i][r0 + m0], a);
#pragma unroll
        for (int m = 0; m < 4; ++m)
          if (m0 + m < i) v[m] = fmaf(-a[m], x[m0 + m], v[m]);
      }
      x[i] = (v[0] + v[1]) + (v[2] + v[3]);
    }
    __syncwarp();
    if (lane < 16) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s.T_[r0 + i][r0 + lane] = x[i];
    }
  }
  __syncthreads();
  // y[0 .. W) of a row of F = (A or T block)[row][m] x G[m][c ..], m < M
  auto block_row = [&](auto& y, int M, const float* frow, float sign, const float* grow, int pitch) {
    constexpr int W = sizeof(y) / sizeof(float);
#pragma unroll 8
    for (int m = 0; m < M; ++m) {
      const float a = sign * frow[m];
#pragma unroll
      for (int e = 0; e < W; e += 4) {
        float x[4];
        load4(grow + m * pitch + e, x);
#pragma unroll
        for (int q = 0; q < 4; ++q) y[e + q] = fmaf(a, x[q], y[e + q]);
      }
    }
  };
  // What is not finite becomes 0, and row r's X NaN (see is_bad): the next product has zeros beside it, above T's diagonal.
  auto finite = [&](auto& y, int r) {
    constexpr int W = sizeof(y) / sizeof(float);
    float big = max3_abs(y[0], y[1], max3_abs(y[2], y[3], 0.0f));
    if constexpr (W == 8) big = max3_abs(big, max3_abs(y[4], y[5], 0.0f), max3_abs(y[6], y[7], 0.0f));
    if (!is_bad(big)) return;
    p.vec[at * kVec + 2 * kC + r] = quiet_nan();
#pragma unroll
    for (int e = 0; e < W; ++e) y[e] = is_bad(y[e]) ? 0.0f : y[e];
  };
  {
    const int pr = 32 * (tid >> 6), r = (tid & 63) >> 2, c = 4 * (tid & 3);
    float y[4] = {}, x[4] = {};
    block_row(y, 16, &s.T_[pr + 16 + r][pr], 1.0f, &s.T_[pr][pr + c], kPitch);
    finite(y, pr + 16 + r);
#pragma unroll
    for (int e = 0; e < 4; ++e) s.tmp[r][(pr >> 1) + c + e] = y[e];
    __syncthreads();
    block_row(x, 16, &s.T_[pr + 16 + r][pr + 16], -1.0f, &s.tmp[0][(pr >> 1) + c], 36);
#pragma unroll
    for (int e = 0; e < 4; ++e) s.T_[pr + 16 + r][pr + c + e] = x[e];
  }
  __syncthreads();
  {
    const int r = tid >> 2, c = 8 * (tid & 3);
    float y[8] = {}, x[8] = {};
    block_row(y, 32, &s.T_[32 + r][0], 1.0f, &s.T_[0][c], kPitch);
    finite(y, 32 + r);
#pragma unroll
    for (int e = 0; e < 8; ++e) s.tmp[r][c + e] = y[e];
    __syncthreads();
    block_row(x, 32, &s.T_[32 + r][32], -1.0f, &s.tmp[0][c], 36);
#pragma unroll
    for (int e = 0; e < 8; ++e) s.T_[32 + r][c + e] = x[e];
  }
  __syncthreads();
#pragma unroll 2
  for (int e = tid; e < kC * kC / 8; e += 128) {
    const int r = e / (kC / 8), grp = e % (kC / 8);
    float x[8];
    load8<float>(s.T_[r], 8 * grp, kC, true, x);
    finite(x, r);
    put_pieces<3>(x, nullptr, p.timg + at * (3 * kTri), tile_off<kC>(r, grp), kTri);
  }
}

// ================================================================================================
// The chain kernels: a CTA carries NS (one or two) strips of 16 value channels of one head's state through all
// chunks, four warps per strip, and one more warp loads the chunks' tiles.  The chain from chunk to chunk is what
// takes the time: it is cut four ways inside a strip (three exchanges per chunk, barriers of four warps), and the
// strips of a CTA run freely, so that one's exchange hides behind another's products.  A chunk takes 2.3 us with
// one strip per SM (bf16, dk 128), of which the tensor pipe is busy 0.7: waits for operands and for one another's
// results bound it.  Where heads are many, ssm_delta_tc.cuh is faster.
// Tiles: K is used first and last in a chunk and has two buffers where they fit, like the vectors; Q, T and P have
// one each, refilled as soon as every strip is past them.
// ================================================================================================
template <typename T, int DKP, int PU, int PO>       // pieces of the operands uf and of
struct alignas(16) StripSmem {
  uint4 sf[DKP / 16][3][32], xf[4][3][32], lf[4][3][32], uf[4][PU][32], of[PO ? 4 : 1][PO ? PO : 1][PO ? 32 : 1];
  Strip<T> in, out;
  int first[2][16];                       // by chunk parity: a channel's first position that is not finite, or kC
  int stop;                               // a wait gave up, as the strip's leader saw it between two barriers
};
template <int NP, int DKP, int PP, typename StripT, int NS, int KB>
struct alignas(128) ChainSmem {
  __nv_bfloat16 k[KB][NP][kC * DKP], q[NP][kC * DKP];
  __nv_bfloat16 t[3][kTri], pm[PP][kTri];
  StripT strip[NS];
  float vec[2][kVec];
  uint64_t full[7], empty[7];             // by tile
  int dead;                               // a wait gave up
};
enum { kTileK = 0, kTileV = 2, kTileQ = 4, kTileT = 5, kTileP = 6, kTiles = 7 };   // K, vectors: two each

// A bounded wait that tells the CTA when it gave up: the strips then stop behind the chunk (z.stop, the same for
// a strip's four warps), and no copy is started any more.  (Asked inside the wait, the flag costs the long prompt 4 %, a flag
// per thread, as in Wait, 12 %.)
template <typename Smem>
__device__ __forceinline__ void chain_wait(Smem& s, uint64_t* bar, uint32_t parity, int* err) {
  for (uint32_t it = 0; it < kPolls; ++it)
    if (mbar_try_wait(bar, parity)) return;
  *static_cast<volatile int*>(&s.dead) = 1;
  if (err) atomicOr(err, 1);
}
// Before the kernel ends: after a wait that gave up, time for its copies in flight to land.
template <typename Smem>
__device__ __forceinline__ void chain_drain(Smem& s) {
  for (int i = 0; *static_cast<volatile int*>(&s.dead) && i < 1000; ++i) __nanosleep(1000);
}

// The tiles of one chunk after another, chunk index by order(i), as the strips release them.
template <int NP, int DKP, int KB, typename Smem, typename F>
__device__ void load_tiles(Smem& s, const DeltaParams& p, int b, int h, F order) {
  const size_t at0 = ((size_t)b * p.Hv + h) * p.n, atk0 = ((size_t)b * p.Hk + h / p.group) * p.n;
  auto freed = [&](int tile, int use) {
    if (use > 0) chain_wait(s, &s.empty[tile], (use - 1) & 1, p.err);
  };
  for (int i = 0; i < p.n && !*static_cast<volatile int*>(&s.dead); ++i) {
    const int ch = order(i);
    auto load_k = [&] {
      const int buf = i % KB, tile = kTileK + buf;
      freed(tile, i / KB);
      mbar_arrive_expect_tx(&s.full[tile], sizeof(s.k[0]));
      bulk_load(s.k[buf], p.kimg + (atk0 + ch) * (NP * kC * DKP), sizeof(s.k[0]), &s.full[tile]);
    };
    freed(kTileV + (i & 1), i >> 1);
    mbar_arrive_expect_tx(&s.full[kTileV + (i & 1)], sizeof(s.vec[0]));
    bulk_load(s.vec[i & 1], p.vec + (at0 + ch) * kVec, sizeof(s.vec[0]), &s.full[kTileV + (i & 1)]);
    if (KB == 2) load_k();
    freed(kTileQ, i);
    mbar_arrive_expect_tx(&s.full[kTileQ], sizeof(s.q));
    bulk_load(s.q, p.qimg + (atk0 + ch) * (NP * kC * DKP), sizeof(s.q), &s.full[kTileQ]);
    if (KB == 1) load_k();
    freed(kTileT, i);
    mbar_arrive_expect_tx(&s.full[kTileT], sizeof(s.t));
    bulk_load(s.t, p.timg + (at0 + ch) * (3 * kTri), sizeof(s.t), &s.full[kTileT]);
    freed(kTileP, i);
    mbar_arrive_expect_tx(&s.full[kTileP], sizeof(s.pm));
    bulk_load(s.pm, p.pimg + (at0 + ch) * (3 * kTri), sizeof(s.pm), &s.full[kTileP]);
  }
  chain_drain(s);
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void strip_sync(int strip) { asm volatile("bar.sync %0, 128;" ::"r"(strip + 1) : "memory"); }

// A quarter of the state (dk, dv) of a head in global memory from / to accumulators of S^T.
template <int NT>
__device__ __forceinline__ void state_load(const float* base, int dk, int dv, int k0, int d0, int lane, float (&S)[NT][4]) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int k = k0 + 8 * j + 2 * t + (e & 1), d = d0 + g + 8 * (e >> 1);
      S[j][e] = base != nullptr && k < dk && d < dv ? base[(size_t)k * dv + d] : 0.0f;
    }
}
template <int NT>
__device__ __forceinline__ void state_store(float* base, int dk, int dv, int k0, int d0, int lane, const float (&S)[NT][4]) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int k = k0 + 8 * j + 2 * t + (e & 1), d = d0 + g + 8 * (e >> 1);
      if (k < dk && d < dv) base[(size_t)k * dv + d] = S[j][e];
    }
}
// The warp's quarter of S in operand form for the strip.
template <int DKP>
__device__ __forceinline__ void put_state(uint4 (*sf)[3][32], const float (&S)[DKP / 32][4], int w, int lane) {
#pragma unroll
  for (int j = 0; j < DKP / 32; j += 2) {
    uint32_t a[3][4];
    acc_to_a<3>(S, j / 2, a);
#pragma unroll
    for (int i = 0; i < 3; ++i)
      sf[(w * (DKP / 32) + j) / 2][i][lane] = make_uint4(a[i][0], a[i][1], a[i][2], a[i][3]);
  }
}

// The warp's two column tiles of d (16 x kC) += S times the transpose of a [c][dk] tile, and, with TWO, of d2
// for a second tile with products up to index sum MAXI2.
template <int NP, int DKP, bool TWO, int MAXI2>
__device__ __forceinline__ void state_product(float (&d)[2][4], float (&d2)[2][4], const uint4 (*sf)[3][32], uint32_t tile,
                                              uint32_t tile2, int w, int lane) {
  float low[2][4], low2[2][4];
  zero(low);
  zero(low2);
#pragma unroll 4
  for (int kb = 0; kb < DKP / 16; ++kb) {
    uint32_t a[3][4];
#pragma unroll
    for (int i = 0; i < 3; ++i) get_frag(a[i], sf[kb][i][lane]);
#pragma unroll
    for (int pb = 0; pb < NP; ++pb) {
      uint32_t bf[1][4], cf[1][4];
      load_b2<DKP>(bf[0], tile + pb * (kC * DKP * 2), w, kb, lane);
      if (TWO && pb <= MAXI2) load_b2<DKP>(cf[0], tile2 + pb * (kC * DKP * 2), w, kb, lane);
      mma_split<2>(d, low, 0, a, bf, pb);
      if (TWO && pb <= MAXI2) mma_split<MAXI2>(d2, low2, 0, a, cf, pb);
    }
  }
  add(d, low);
  if (TWO) add(d2, low2);
}

// The warp's two column tiles of a product with a triangular kC x kC tile: d[.][i] += sum_k a[.][k] L[i][k] (TR
// false, L lower: k blocks up to the column's) or d[.][j] += sum_i a[.][i] L[i][j] (TR true: k blocks from it).
// a: the strip's operand in NA pieces; products up to index sum MAXI.
template <int NA, int NB, int MAXI, bool TR>
__device__ __forceinline__ void tri_product(float (&d)[2][4], const uint4 (*f)[NA][32], uint32_t tile, int w, int lane) {
  float low[3][2][4];                    // by piece of the tile: six chains of products instead of two
#pragma unroll
  for (int pb = 0; pb < 3; ++pb) zero(low[pb]);
#pragma unroll
  for (int kb = 0; kb < kC / 16; ++kb) {
    const bool first = TR ? 2 * kb + 1 >= w : 2 * kb <= w;             // whether the tiles w and 7 - w need kb
    const bool second = TR ? 2 * kb + 1 >= 7 - w : 2 * kb <= 7 - w;
    if (!first && !second) continue;
    uint32_t a[NA][4], bf[NB][4];
#pragma unroll
    for (int i = 0; i < NA; ++i) get_frag(a[i], f[kb][i][lane]);
#pragma unroll
    for (int pb = 0; pb < NB && pb <= MAXI; ++pb) {
      if (TR) load_bt2<kC>(bf[pb], tile + pb * (kTri * 2), w, kb, lane);
      else load_b2<kC>(bf[pb], tile + pb * (kTri * 2), w, kb, lane);
    }
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
      for (int pb = 0; pb < NB; ++pb) {
        if (i + pb > MAXI) continue;
        if (first) mma_bf16(i + pb ? low[pb][0] : d[0], a[i], bf[pb][0], bf[pb][1]);
        if (second) mma_bf16(i + pb ? low[pb][1] : d[1], a[i], bf[pb][2], bf[pb][3]);
      }
  }
#pragma unroll
  for (int pb = 0; pb < NB && pb <= MAXI; ++pb) add(d, low[pb]);
}

// The warp's quarter of S <- decay S + sign (a [.][c]) (tile [c][dk]) over kC positions.  The sum over the chunk is
// formed on its own and added once, rounded to nearest: a state that the tensor cores accumulated over
// hundreds of chunks, truncating each time, would drift.
template <int NP, int DKP>
__device__ __forceinline__ void state_add(float (&S)[DKP / 32][4], float2 decay, float sign, const uint4 (*f)[3][32],
                                          uint32_t tile, int w, int lane) {
  constexpr int NT = DKP / 32;
  float d[NT][4], low[NT][4];
  zero(d);
  zero(low);
#pragma unroll
  for (int kb = 0; kb < kC / 16; ++kb) {
    uint32_t a[3][4];
#pragma unroll
    for (int i = 0; i < 3; ++i) get_frag(a[i], f[kb][i][lane]);
#pragma unroll
    for (int pb = 0; pb < NP; ++pb) {
      uint32_t bf[NT / 2][4];
#pragma unroll
      for (int j = 0; j < NT / 2; ++j) load_bt<DKP>(bf[j], tile + pb * (kC * DKP * 2), w * NT + 2 * j, kb, lane);
      mma_split<2>(d, low, 0, a, bf, pb);
    }
  }
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) S[j][e] = fmaf(e >> 1 ? decay.y : decay.x, S[j][e], sign * (d[j][e] + low[j][e]));
}

// The per-position factors of the columns 2 t, 2 t + 1 of a column tile.
__device__ __forceinline__ float2 at_cols(const float* v, int tile, int t) {
  return *reinterpret_cast<const float2*>(v + 8 * tile + 2 * t);
}
// The warp's column tiles of a dense fp32 [channel][kC] block.
__device__ __forceinline__ void store_cols(float* base, int w, int lane, const float (&c)[2][4]) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float* o = base + g * kC + 8 * col_tile(w, j) + 2 * t;
    *reinterpret_cast<float2*>(o) = make_float2(c[j][0], c[j][1]);
    *reinterpret_cast<float2*>(o + 8 * kC) = make_float2(c[j][2], c[j][3]);
  }
}
// See is_bad: values of the warp's column tiles, positions by column, channels by row.  What is not finite becomes 0 and is
// noted in `first`, by channel.
__device__ __forceinline__ void note_bad(float (&x)[2][4], int* first, int w, int lane) {
  const float big = max3_abs(max3_abs(x[0][0], x[0][1], x[0][2]), max3_abs(x[0][3], x[1][0], x[1][1]), max3_abs(x[1][2], x[1][3], 0.0f));
  if (!is_bad(big)) return;
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (is_bad(x[j][e])) {
        atomicMin(first + (lane >> 2) + 8 * (e >> 1), 8 * col_tile(w, j) + 2 * (lane & 3) + (e & 1));
        x[j][e] = 0.0f;
      }
}
// NaN from a channel's first position that is not finite.
__device__ __forceinline__ void set_from(float (&x)[2][4], const int* first, int w, int lane) {
  const int f0 = first[lane >> 2], f1 = first[(lane >> 2) + 8];
  if (min(f0, f1) >= kC) return;
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (8 * col_tile(w, j) + 2 * (lane & 3) + (e & 1) >= (e >> 1 ? f1 : f0)) x[j][e] = quiet_nan();
}
template <typename Smem>
__device__ __forceinline__ void init_tiles(Smem& s, int strips) {
  if (threadIdx.x == 0) {
    for (int i = 0; i < kTiles; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], strips);
    }
    s.dead = 0;
    fence_mbar_init();
  }
  __syncthreads();
}

template <typename T, int NP, int DKP, int NS>
struct FwdChain {
  // Pieces of P and of its U (and index sums of Q S): a bf16 o is kept to 16 bits before it is rounded to 8.  One value in 400
  // then rounds the other way than from 24 bits; o's error against 64 bits is that rounding's, 1.659e-3, either way.
  static constexpr int PP = NP == 1 ? 2 : 3;
  using StripT = StripSmem<T, DKP, PP, 0>;
  template <int KB>
  using Smem = ChainSmem<NP, DKP, PP, StripT, NS, KB>;
  static constexpr int KB = sizeof(Smem<2>) <= 227 * 1024 ? 2 : 1;
};
template <typename T, int NP, int DKP, int NS>
struct BwdChain {
  using StripT = StripSmem<T, DKP, 3, NP>;
  template <int KB>
  using Smem = ChainSmem<NP, DKP, 3, StripT, NS, KB>;
  static constexpr int KB = sizeof(Smem<2>) <= 227 * 1024 ? 2 : 1;
};

// CTAs that shared memory lets on an SM: registers are shared out accordingly (the compiler's own choice, 128 a thread, made the
// long prompt 3 % slower).
template <int NP, int DKP, int NS>
constexpr int kChainCtas = NP == 1 && DKP == 64 && NS == 1 ? 2 : 1;

// ================================================================================================
// Forward chain
// ================================================================================================
template <typename T, int NP, int DKP, int NS, bool SAVE>
__global__ void __launch_bounds__(128 * NS + 32, kChainCtas<NP, DKP, NS>) delta_fwd(const __grid_constant__ DeltaParams p) {
  using Form = FwdChain<T, NP, DKP, NS>;
  constexpr int PP = Form::PP, KB = Form::KB, NT = DKP / 32;
  using Smem = typename Form::template Smem<KB>;
  extern __shared__ __align__(128) unsigned char smem_raw[];
  Smem& s = *reinterpret_cast<Smem*>(smem_raw);
  const int strip = threadIdx.x >> 7, w = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31, t = lane & 3;
  const int h = blockIdx.y, b = blockIdx.z;
  const int strips = min(NS, p.dvp / 16 - (int)blockIdx.x * NS);
  init_tiles(s, strips);
  if (strip >= NS) {
    if (lane == 0) load_tiles<NP, DKP, KB>(s, p, b, h, [](int i) { return i; });
    return;
  }
  if (strip >= strips) return;
  const int d0 = 16 * (blockIdx.x * NS + strip), cols = p.dvw - d0;
  auto& z = s.strip[strip];
  const size_t head = (size_t)b * p.Hv + h;
  float S[NT][4];
  state_load(p.h0 != nullptr ? p.h0 + head * p.dkw * p.dvw : nullptr, p.dkw, p.dvw, 8 * NT * w, d0, lane, S);
  const uint32_t sq = smem_u32(s.q[0]), stt = smem_u32(s.t[0]), sp = smem_u32(s.pm[0]);
  const T* vbase = static_cast<const T*>(p.v.ptr) + b * p.v.sb + h * p.v.sh + d0;
  T* obase = static_cast<T*>(const_cast<void*>(p.o.ptr)) + b * p.o.sb + h * p.o.sh + d0;
  const bool vin = rows_aligned16(p.v, sizeof(T)), oout = rows_aligned16(p.o, sizeof(T));
  const bool leader = w == 0 && lane == 0;
  if (w == 0) z.first[lane >> 4][lane & 15] = kC;
  z.in.fetch(vbase, p.v.sl, min(kC, p.L), cols, vin, w, lane);
  for (int ch = 0; ch < p.n; ++ch) {
    const int buf = ch % KB, rows = min(kC, p.L - ch * kC);
    const long long t0 = (long long)ch * kC;
    const float* vec = s.vec[ch & 1];
    const uint32_t sk = smem_u32(s.k[buf][0]);
    put_state<DKP>(z.sf, S, w, lane);
    if (SAVE) store_acc(p.states + ((head * p.n + ch) * p.dvp + d0) * DKP + 8 * NT * w, DKP, lane, S);
    strip_sync(strip);                            // S is there; the last chunk is done with
    if (leader) *static_cast<volatile int*>(&z.stop) = *static_cast<volatile int*>(&s.dead);
    if (leader && ch > 0) {
      mbar_arrive(&s.empty[kTileP]);
      mbar_arrive(&s.empty[kTileK + (ch - 1) % KB]);
      mbar_arrive(&s.empty[kTileV + ((ch - 1) & 1)]);
    }
    int* first = z.first[ch & 1];
    if (w == 0 && lane < 16) z.first[(ch + 1) & 1][lane] = kC;
    float V[2][4], X[2][4], O[2][4], U[2][4];
    z.in.arrive();
    z.in.read(V, w, lane);
    __syncwarp();
    if (ch + 1 < p.n)
      z.in.fetch(vbase + (t0 + kC) * p.v.sl, p.v.sl, min(kC, p.L - (ch + 1) * kC), cols, vin, w, lane);
    zero(X);
    zero(O);
    zero(U);
    chain_wait(s, &s.full[kTileK + buf], (ch / KB) & 1, p.err);
    chain_wait(s, &s.full[kTileV + (ch & 1)], (ch >> 1) & 1, p.err);
    chain_wait(s, &s.full[kTileQ], ch & 1, p.err);
    state_product<NP, DKP, true, PP - 1>(X, O, z.sf, sk, sq, w, lane);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float2 eg = at_cols(vec, col_tile(w, j), t), be = at_cols(vec + 2 * kC, col_tile(w, j), t);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float eg_ = e & 1 ? eg.y : eg.x;
        X[j][e] = (e & 1 ? be.y : be.x) * fmaf(-eg_, X[j][e], V[j][e]);
        O[j][e] *= p.scale * eg_;
      }
    }
    note_bad(X, first, w, lane);
#pragma unroll
    for (int j = 0; j < 2; ++j) put_half<3>(z.xf, col_tile(w, j), X[j], lane);
    strip_sync(strip);                            // X is there; Q is done with
    if (leader) mbar_arrive(&s.empty[kTileQ]);
    chain_wait(s, &s.full[kTileT], ch & 1, p.err);
    tri_product<3, 3, 2, false>(U, z.xf, stt, w, lane);
    if (SAVE) {
#pragma unroll
      for (int j = 0; j < 2; ++j) put_half<PP>(z.uf, col_tile(w, j), U[j], lane);
      set_from(U, first, w, lane);
      store_cols(p.us + ((head * p.n + ch) * p.dvp + d0) * kC, w, lane, U);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (!SAVE) put_half<PP>(z.uf, col_tile(w, j), U[j], lane);
      const float2 la = at_cols(vec + kC, col_tile(w, j), t);
#pragma unroll
      for (int e = 0; e < 4; ++e) U[j][e] *= e & 1 ? la.y : la.x;
      put_half<3>(z.lf, col_tile(w, j), U[j], lane);
    }
    strip_sync(strip);                            // U is there; T is done with
    const int f0 = first[lane >> 2], f1 = first[(lane >> 2) + 8];
    if (leader) mbar_arrive(&s.empty[kTileT]);
    chain_wait(s, &s.full[kTileP], ch & 1, p.err);
    tri_product<PP, PP, PP - 1, false>(O, z.uf, sp, w, lane);
    state_add<NP, DKP>(S, make_float2(f0 < kC ? quiet_nan() : vec[kC - 1], f1 < kC ? quiet_nan() : vec[kC - 1]), 1.0f, z.lf, sk, w, lane);
    const int stop = *static_cast<volatile int*>(&z.stop);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        O[j][e] = 8 * col_tile(w, j) + 2 * t + (e & 1) >= (e >> 1 ? f1 : f0) ? quiet_nan() : O[j][e];
    z.out.write(O, w, lane);
    z.out.flush(obase + t0 * p.o.sl, p.o.sl, rows, cols, oout, w, lane);
    if (stop) break;
  }
  if (p.last != nullptr) state_store(p.last + head * p.dkw * p.dvw, p.dkw, p.dvw, 8 * NT * w, d0, lane, S);
  chain_drain(s);
}

// ================================================================================================
// Backward chain, chunks in reverse, with dS' the gradient of the state leaving the chunk:
//   Y = e^(G_last - G) K dS' + P^T dO,  dX = T^T Y,  dV = beta dX
//   dS = e^G_last dS' + (scale e^G Q)^T dO - (beta e^G K)^T dX
// ================================================================================================
template <typename T, int NP, int DKP, int NS>
__global__ void __launch_bounds__(128 * NS + 32, kChainCtas<NP, DKP, NS>) delta_bwd_chain(const __grid_constant__ DeltaParams p) {
  using Form = BwdChain<T, NP, DKP, NS>;
  constexpr int KB = Form::KB, NT = DKP / 32;
  using Smem = typename Form::template Smem<KB>;
  extern __shared__ __align__(128) unsigned char smem_raw[];
  Smem& s = *reinterpret_cast<Smem*>(smem_raw);
  const int strip = threadIdx.x >> 7, w = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31, t = lane & 3;
  const int h = blockIdx.y, b = blockIdx.z;
  const int strips = min(NS, p.dvp / 16 - (int)blockIdx.x * NS);
  init_tiles(s, strips);
  if (strip >= NS) {
    const int last = p.n - 1;
    if (lane == 0) load_tiles<NP, DKP, KB>(s, p, b, h, [last](int i) { return last - i; });
    return;
  }
  if (strip >= strips) return;
  const int d0 = 16 * (blockIdx.x * NS + strip), cols = p.dvw - d0;
  auto& z = s.strip[strip];
  const size_t head = (size_t)b * p.Hv + h;
  float S[NT][4];
  state_load(p.h0 != nullptr ? p.h0 + head * p.dkw * p.dvw : nullptr, p.dkw, p.dvw, 8 * NT * w, d0, lane, S);
  const uint32_t sq = smem_u32(s.q[0]), stt = smem_u32(s.t[0]), sp = smem_u32(s.pm[0]);
  const T* gbase = static_cast<const T*>(p.o.ptr) + b * p.o.sb + h * p.o.sh + d0;
  T* obase = static_cast<T*>(const_cast<void*>(p.dv.ptr)) + b * p.dv.sb + h * p.dv.sh + d0;
  const bool gin = rows_aligned16(p.o, sizeof(T)), oout = rows_aligned16(p.dv, sizeof(T));
  const bool leader = w == 0 && lane == 0;
  z.in.fetch(gbase + (long long)(p.n - 1) * kC * p.o.sl, p.o.sl, p.L - (p.n - 1) * kC, cols, gin, w, lane);
  for (int it = 0; it < p.n; ++it) {
    const int ch = p.n - 1 - it, buf = it % KB, rows = min(kC, p.L - ch * kC);
    const long long t0 = (long long)ch * kC;
    const float* vec = s.vec[it & 1];
    const uint32_t sk = smem_u32(s.k[buf][0]);
    put_state<DKP>(z.sf, S, w, lane);
    store_acc(p.dstates + ((head * p.n + ch) * p.dvp + d0) * DKP + 8 * NT * w, DKP, lane, S);
    float dO[2][4], Y[2][4], X[2][4];
    z.in.arrive();
    z.in.read(dO, w, lane);
    __syncwarp();
    if (ch > 0) z.in.fetch(gbase + (t0 - kC) * p.o.sl, p.o.sl, kC, cols, gin, w, lane);
    chain_wait(s, &s.full[kTileV + (it & 1)], (it >> 1) & 1, p.err);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      put_half<NP>(z.of, col_tile(w, j), dO[j], lane);
      const float2 eg = at_cols(vec, col_tile(w, j), t);
#pragma unroll
      for (int e = 0; e < 4; ++e) dO[j][e] *= p.scale * (e & 1 ? eg.y : eg.x);
      put_half<3>(z.uf, col_tile(w, j), dO[j], lane);
    }
    zero(X);
    zero(Y);
    strip_sync(strip);                            // dS' and dO are there; the last chunk is done with
    if (leader) *static_cast<volatile int*>(&z.stop) = *static_cast<volatile int*>(&s.dead);
    if (leader && it > 0) {
      mbar_arrive(&s.empty[kTileK + (it - 1) % KB]);
      mbar_arrive(&s.empty[kTileV + ((it - 1) & 1)]);
    }
    chain_wait(s, &s.full[kTileK + buf], (it / KB) & 1, p.err);
    state_product<NP, DKP, false, 0>(Y, Y, z.sf, sk, sk, w, lane);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float2 la = at_cols(vec + kC, col_tile(w, j), t);
#pragma unroll
      for (int e = 0; e < 4; ++e) Y[j][e] *= e & 1 ? la.y : la.x;
    }
    chain_wait(s, &s.full[kTileP], it & 1, p.err);
    tri_product<NP, 3, 2, true>(Y, z.of, sp, w, lane);
#pragma unroll
    for (int j = 0; j < 2; ++j) put_half<3>(z.xf, col_tile(w, j), Y[j], lane);
    chain_wait(s, &s.full[kTileQ], it & 1, p.err);
    state_add<NP, DKP>(S, make_float2(vec[kC - 1], vec[kC - 1]), 1.0f, z.uf, sq, w, lane);
    strip_sync(strip);                            // Y is there; P and Q are done with
    if (leader) {
      mbar_arrive(&s.empty[kTileQ]);
      mbar_arrive(&s.empty[kTileP]);
    }
    chain_wait(s, &s.full[kTileT], it & 1, p.err);
    tri_product<3, 3, 2, true>(X, z.xf, stt, w, lane);
    store_cols(p.dxs + ((head * p.n + ch) * p.dvp + d0) * kC, w, lane, X);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float2 eg = at_cols(vec, col_tile(w, j), t), be = at_cols(vec + 2 * kC, col_tile(w, j), t);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        Y[j][e] = X[j][e] * (e & 1 ? be.y : be.x);
        X[j][e] = Y[j][e] * (e & 1 ? eg.y : eg.x);
      }
      put_half<3>(z.lf, col_tile(w, j), X[j], lane);
    }
    strip_sync(strip);                            // dX is there; T is done with
    if (leader) mbar_arrive(&s.empty[kTileT]);
    state_add<NP, DKP>(S, make_float2(1.0f, 1.0f), -1.0f, z.lf, sk, w, lane);
    const int stop = *static_cast<volatile int*>(&z.stop);
    z.out.write(Y, w, lane);
    z.out.flush(obase + t0 * p.dv.sl, p.dv.sl, rows, cols, oout, w, lane);
    if (stop) break;
  }
  if (p.last != nullptr) state_store(p.last + head * p.dkw * p.dvw, p.dkw, p.dvw, 8 * NT * w, d0, lane, S);
  chain_drain(s);
}

// dq, dk (B, L, Hk, dk): the value heads' parts, (B, L, Hv, DKP) fp32, summed in head order.  A thread takes four
// channels of one position and key head (blockIdx.x walks positions, blockIdx.y key heads).  Memory bounds it: 8192
// positions x 40 heads of 128 in 72 us, 5.8 TB/s.
template <typename T, int DKP>
__global__ void __launch_bounds__(256) delta_sum_heads(const __grid_constant__ DeltaParams p) {
  constexpr int kPer = 256 / (DKP / 4);              // positions per CTA
  const int c = 4 * (threadIdx.x % (DKP / 4)), hk = blockIdx.y;
  const long long row = (long long)blockIdx.x * kPer + threadIdx.x / (DKP / 4);
  if (row >= (long long)p.B * p.L || c >= p.dkw) return;
  const long long b = row / p.L, l = row - b * p.L;
  float dq[4] = {}, dk[4] = {};
  for (int r = 0; r < p.group; ++r) {
    const size_t o = ((size_t)row * p.Hv + hk * p.group + r) * DKP + c;
    float x[4], y[4];
    load4(p.pdq + o, x);
    load4(p.pdk + o, y);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      dq[e] += x[e];
      dk[e] += y[e];
    }
  }
  T* dqp = static_cast<T*>(const_cast<void*>(p.dq.ptr)) + b * p.dq.sb + l * p.dq.sl + hk * p.dq.sh + c;
  T* dkp = static_cast<T*>(const_cast<void*>(p.dk.ptr)) + b * p.dk.sb + l * p.dk.sl + hk * p.dk.sh + c;
  constexpr int kBytes = 4 * (int)sizeof(T);
  if (c + 4 <= p.dkw && ((reinterpret_cast<uintptr_t>(dqp) | reinterpret_cast<uintptr_t>(dkp)) & (kBytes - 1)) == 0) {
    vec_store<T, 4>(dqp, dq);
    vec_store<T, 4>(dkp, dk);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < p.dkw) {
        dqp[e] = from_f32<T>(dq[e]);
        dkp[e] = from_f32<T>(dk[e]);
      }
  }
}

// ================================================================================================
// One token: S <- a S, e = beta (v - S^T k), S <- S + k e^T, o = scale S^T q.
// A CTA of eight warps takes 32 VEC value channels of one head: a lane has VEC of them, a warp every eighth row
// of dk, ROWS in all.  The rows stay in registers between the two passes over them, so the state is read and
// written once, which bounds the kernel: 64 x 16 heads of 128 x 128 in 23 us, 5.8 TB/s (one channel a lane: 44 us).
// ================================================================================================
template <typename T, int VEC, int ROWS>
__global__ void __launch_bounds__(256) delta_step(const __grid_constant__ DeltaParams p) {
  __shared__ float red[2][8][32 * VEC], kq[2][8 * ROWS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h = blockIdx.y, b = blockIdx.z, hk = h / p.group;
  const int d = (blockIdx.x * 32 + lane) * VEC;
  const bool live = d < p.dvw;
  float* S = p.last + ((size_t)b * p.Hv + h) * p.dkw * p.dvw + d;
  float x[ROWS][VEC], part[VEC], e[VEC];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int r = warp + 8 * i;
#pragma unroll
    for (int v = 0; v < VEC; ++v) x[i][v] = 0.0f;
    if (live && r < p.dkw) vec_load<float, VEC>(S + (size_t)r * p.dvw, x[i]);
  }
  const float alpha = expf(p.g[b * p.gsb + h]), beta = p.beta[b * p.bsb + h];
  for (int i = threadIdx.x; i < 16 * ROWS; i += 256) {
    const int which = i / (8 * ROWS), r = i % (8 * ROWS);
    const Heads& src = which ? p.q : p.k;
    kq[which][r] = r < p.dkw ? to_f32(static_cast<const T*>(src.ptr)[b * src.sb + hk * src.sh + r]) : 0.0f;
  }
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    part[v] = 0.0f;
    e[v] = live ? to_f32(static_cast<const T*>(p.v.ptr)[b * p.v.sb + h * p.v.sh + d + v]) : 0.0f;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const float k = kq[0][warp + 8 * i];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      x[i][v] *= alpha;
      part[v] = fmaf(x[i][v], k, part[v]);
    }
  }
  vec_store<float, VEC>(&red[0][warp][lane * VEC], part);
  __syncthreads();
  float dot[VEC] = {};
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    float y[VEC];
    vec_load<float, VEC>(&red[0][w][lane * VEC], y);
#pragma unroll
    for (int v = 0; v < VEC; ++v) dot[v] += y[v];
  }
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    e[v] = beta * (e[v] - dot[v]);
    part[v] = 0.0f;
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int r = warp + 8 * i;
    const float k = kq[0][r], q = kq[1][r];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      x[i][v] = fmaf(k, e[v], x[i][v]);
      part[v] = fmaf(x[i][v], q, part[v]);
    }
    if (live && r < p.dkw) vec_store<float, VEC>(S + (size_t)r * p.dvw, x[i]);
  }
  vec_store<float, VEC>(&red[1][warp][lane * VEC], part);
  __syncthreads();
  if (warp == 0 && live) {
    T* o = static_cast<T*>(const_cast<void*>(p.o.ptr)) + b * p.o.sb + h * p.o.sh + d;
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < 8; ++w) s += red[1][w][lane * VEC + v];
      o[v] = from_f32<T>(p.scale * s);
    }
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
  if (s.B > 65535 || s.Hv > 65535 || s.dv > (1 << 20) || s.L > (1LL << 30) || s.B * s.Hv * s.n() > (1LL << 31) - 1024)
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

// The parts of a buffer; with base null only its size is of use.  Everything delta_prep writes:
void carve_prep(const Shape& s, DeltaParams& p, Carver& c) {
  const size_t chunks_k = (size_t)s.B * s.Hk * s.n(), chunks = (size_t)s.B * s.Hv * s.n();
  p.kimg = c.take<__nv_bfloat16>(chunks_k * s.np() * kC * s.dkp());
  p.qimg = c.take<__nv_bfloat16>(chunks_k * s.np() * kC * s.dkp());
  p.timg = c.take<__nv_bfloat16>(chunks * 3 * kTri);
  p.pimg = c.take<__nv_bfloat16>(chunks * 3 * kTri);
  p.vec = c.take<float>(chunks * kVec);
}
// What a training forward leaves for the backward: that (again computing it took 10 % of a training pass), the
// states and the corrected values.
size_t carve_saved(const Shape& s, DeltaParams& p, unsigned char* base) {
  Carver c{base};
  carve_prep(s, p, c);
  const size_t chunks = (size_t)s.B * s.Hv * s.n();
  p.states = c.take<float>(chunks * s.dvp() * s.dkp());
  p.us = c.take<float>(chunks * s.dvp() * kC);
  return c.used + 256;
}
size_t carve_fwd(const Shape& s, DeltaParams& p, unsigned char* base) {
  Carver c{base};
  carve_prep(s, p, c);
  return c.used + 256;
}
size_t carve_bwd(const Shape& s, DeltaParams& p, unsigned char* base) {
  Carver c{base};
  const size_t chunks = (size_t)s.B * s.Hv * s.n();
  p.dstates = c.take<float>(chunks * s.dvp() * s.dkp());
  p.dxs = c.take<float>(chunks * s.dvp() * kC);
  if (s.Hv > s.Hk) {
    p.pdq = c.take<float>((size_t)s.B * s.L * s.Hv * s.dkp());
    p.pdk = c.take<float>((size_t)s.B * s.L * s.Hv * s.dkp());
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

template <auto Kern>
cudaError_t launch(dim3 grid, int threads, size_t smem, const DeltaParams& p, cudaStream_t st) {
  if (smem > 48 * 1024) ctas_per_sm<Kern>(threads, smem);
  Kern<<<grid, threads, smem, st>>>(p);
  return cudaGetLastError();
}

template <typename T, int NP, int DKP, int NS>
cudaError_t run_chain_ns(const Shape& s, const DeltaParams& p, bool bwd, cudaStream_t st) {
  const dim3 grid((unsigned)((s.dvp() / 16 + NS - 1) / NS), (unsigned)s.Hv, (unsigned)s.B);
  constexpr int threads = 128 * NS + 32;
  if (bwd) {
    using Form = BwdChain<T, NP, DKP, NS>;
    constexpr size_t smem = sizeof(typename Form::template Smem<Form::KB>);
    static_assert(smem <= 227 * 1024, "shared memory");
    return launch<delta_bwd_chain<T, NP, DKP, NS>>(grid, threads, smem, p, st);
  } else {
    using Form = FwdChain<T, NP, DKP, NS>;
    constexpr size_t smem = sizeof(typename Form::template Smem<Form::KB>);
    static_assert(smem <= 227 * 1024, "shared memory");
    return p.states != nullptr ? launch<delta_fwd<T, NP, DKP, NS, true>>(grid, threads, smem, p, st)
                               : launch<delta_fwd<T, NP, DKP, NS, false>>(grid, threads, smem, p, st);
  }
}
template <typename T, int NP, int DKP>
cudaError_t run_chain_tc(const Shape& s, const DeltaParams& p, bool bwd, cudaStream_t st) {
  const dim3 grid((unsigned)((s.dv + 127) / 128), (unsigned)s.Hv, (unsigned)s.B);
  constexpr size_t fwd = sizeof(TcSmem<NP, DKP, NP == 1 ? 2 : 3>) + 1024, back = sizeof(TcSmem<NP, DKP, 3>) + 1024;
  static_assert(back <= 227 * 1024, "two stages of tiles");
  if (bwd) return launch<delta_bwd_tc<T, NP, DKP>>(grid, kTcThreads, back, p, st);
  return p.states != nullptr ? launch<delta_fwd_tc<T, NP, DKP, true>>(grid, kTcThreads, fwd, p, st)
                             : launch<delta_fwd_tc<T, NP, DKP, false>>(grid, kTcThreads, fwd, p, st);
}
// Which chain kernel: strips, one or two to a CTA, or tcgen05.  One CTA of each fills an SM's shared memory (of the bf16 ones
// with one strip and dk up to 64, two do), so a call takes waves of 148 CTAs.  What a wave takes was measured over 4 to
// 1184 strips in 4 to 385 heads (us for 1024 positions, 1965 MHz; forward, the mean of inference and training / backward):
//                         bf16, dk 128     bf16, dk 64                    fp32, dk 64
//   one strip             41 / 48          46 / 54 (up to 148: 40 / 43)   43 / 50
//   two strips            60 / 69          47 / 55                        64 / 68
//   tcgen05, 128 rows     112 / 121        84 / 99                        115 / 122
// Heads with an odd number of strips give CTAs of two and of one: about the work's share of 148 SMs and half a pair more, unless
// all run at once.  By this, the slowest of 198 choices is 8 % behind the best of the three measured, six are over 6 %.  Two
// strips never pay in bf16 at dk 64; fp32 keys above 64 channels leave shared memory for one strip only.
// Returns the value channels that a CTA takes: 16 or 32 (strips), 128 (tcgen05).
int chain_rows(const Shape& s, bool bwd) {
  const bool wide = s.dkp() == 128, f32 = s.np() == 3;
  if (f32 && wide) return 16;
  const int64_t heads = s.B * s.Hv, strips = s.dvp() / 16, pairs = (strips + 1) / 2;
  auto waves = [heads](int64_t ctas_per_head) { return (double)((heads * ctas_per_head + 147) / 148); };
  const double tc = waves((s.dv + 127) / 128) * (wide ? (bwd ? 121 : 112) : f32 ? (bwd ? 122 : 115) : (bwd ? 99 : 84));
  if (!wide && !f32) {
    const int64_t full = heads * strips / 296, rest = heads * strips % 296;
    const double wave = bwd ? 54 : 46;
    const double one = (double)full * wave + (rest == 0 ? 0.0 : rest > 148 ? wave : bwd ? 43.0 : 40.0);
    return tc < one ? 128 : 16;
  }
  const double strip = wide ? (bwd ? 48 : 41) : (bwd ? 50 : 43), pair = wide ? (bwd ? 69 : 60) : (bwd ? 68 : 64);
  const double one = waves(strips) * strip;
  double two = waves(pairs) * pair;
  if (strips == 1) two = one;
  else if (strips % 2 != 0 && heads * pairs > 148)
    two = (double)heads * ((double)(strips / 2) * pair + strip) / 148.0 + 0.5 * pair;
  if (tc < one && tc < two) return 128;
  return two < one ? 32 : 16;
}
template <typename T, int NP, int DKP>
cudaError_t run_chain(const Shape& s, const DeltaParams& p, bool bwd, cudaStream_t st) {
  if constexpr (NP == 1 || DKP == 64) {
    const int rows = chain_rows(s, bwd);
    if (rows == 128) return run_chain_tc<T, NP, DKP>(s, p, bwd, st);
    if constexpr (NP == 3 || DKP == 128)
      if (rows == 32) return run_chain_ns<T, NP, DKP, 2>(s, p, bwd, st);
  }
  return run_chain_ns<T, NP, DKP, 1>(s, p, bwd, st);
}
template <typename T, int NP, int DKP>
cudaError_t run_fwd(const Shape& s, const DeltaParams& p, cudaStream_t st) {
  const dim3 grid((unsigned)s.n(), (unsigned)s.Hv, (unsigned)s.B);
  const cudaError_t e = launch<delta_prep<T, NP, DKP>>(grid, 128, sizeof(PrepSmem<NP, DKP>), p, st);
  return e != cudaSuccess ? e : run_chain<T, NP, DKP>(s, p, false, st);
}

template <typename T, int NP, int DKP>
cudaError_t run_bwd(const Shape& s, const DeltaParams& p, cudaStream_t st) {
  cudaError_t e = run_chain<T, NP, DKP>(s, p, true, st);
  if (e != cudaSuccess) return e;
  const dim3 bg((unsigned)std::min<int64_t>(s.n() * s.Hv * s.B, 148));       // one CTA per SM walks over the chunks
  constexpr size_t smem = sizeof(ChunkSmem<NP, DKP>) + 1024;
  static_assert(smem <= 227 * 1024 && smem > 114 * 1024, "one CTA per SM, which takes all tensor memory");
  e = launch<delta_bwd_chunk<T, NP, DKP>>(bg, kChunkThreads, smem, p, st);
  if (e != cudaSuccess || p.group == 1) return e;
  constexpr int per = 256 / (DKP / 4);
  const dim3 sg((unsigned)(((long long)p.B * p.L + per - 1) / per), (unsigned)p.Hk);
  return launch<delta_sum_heads<T, DKP>>(sg, 256, 0, p, st);
}

// Four value channels a lane (16-byte accesses) where the state's rows allow it and that still gives every SM a CTA,
// else one, in four times the CTAs.
template <typename T>
cudaError_t run_step(const Shape& s, const DeltaParams& p, cudaStream_t st) {
  const bool aligned = s.dv % 4 == 0 && reinterpret_cast<uintptr_t>(p.last) % 16 == 0;
  const bool wide = aligned && s.B * s.Hv * ((s.dv + 127) / 128) >= 148;
  const int per = wide ? 128 : 32;
  const dim3 grid((unsigned)((s.dv + per - 1) / per), (unsigned)s.Hv, (unsigned)s.B);
  if (s.dk <= 64)
    return wide ? launch<delta_step<T, 4, 8>>(grid, 256, 0, p, st) : launch<delta_step<T, 1, 8>>(grid, 256, 0, p, st);
  return wide ? launch<delta_step<T, 4, 16>>(grid, 256, 0, p, st) : launch<delta_step<T, 1, 16>>(grid, 256, 0, p, st);
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
  memset(&p, 0, sizeof(p));
  *bytes = backward ? carve_bwd(s, p, nullptr) : carve_fwd(s, p, nullptr);
  return SSM_OK;
}

int ssm_gated_delta_saved_size(int64_t B, int64_t L, int64_t Hk, int64_t Hv, int64_t dk, int64_t dv, int32_t dtype,
                               size_t* bytes) {
  if (bytes == nullptr) return fail(SSM_ERR_INVALID, "gated delta rule: bytes is NULL");
  const Shape s{B, L, Hk, Hv, dk, dv, dtype};
  int rc = check_shape(s);
  if (rc) return rc;
  DeltaParams p;
  memset(&p, 0, sizeof(p));
  *bytes = carve_saved(s, p, nullptr);
  return SSM_OK;
}

int ssm_gated_delta_plan(int64_t B, int64_t L, int64_t Hk, int64_t Hv, int64_t dk, int64_t dv, int32_t dtype,
                         int32_t backward, int32_t* channels) {
  if (channels == nullptr) return fail(SSM_ERR_INVALID, "gated delta rule: channels is NULL");
  const Shape s{B, L, Hk, Hv, dk, dv, dtype};
  int rc = check_shape(s);
  if (rc) return rc;
  *channels = chain_rows(s, backward != 0);
  return SSM_OK;
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
  if (saved != nullptr) {          // a training call needs no workspace beside it
    carve_saved(s, p, align256(saved));
  } else {
    const size_t need = carve_fwd(s, p, nullptr);
    if (workspace == nullptr || workspace_bytes < need)
      return fail(SSM_ERR_WORKSPACE, "gated delta rule: forward workspace of %zu bytes required, %zu given", need,
                  workspace_bytes);
    carve_fwd(s, p, align256(workspace));
  }
  fill(p, s, q, k, v, g, beta, scale);
  p.o = heads(o);
  p.h0 = h0;
  p.last = last;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (s.dtype == SSM_BF16)
    e = s.dkp() == 64 ? run_fwd<__nv_bfloat16, 1, 64>(s, p, st)
                      : run_fwd<__nv_bfloat16, 1, 128>(s, p, st);
  else
    e = s.dkp() == 64 ? run_fwd<float, 3, 64>(s, p, st)
                      : run_fwd<float, 3, 128>(s, p, st);
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
  const size_t need = carve_bwd(s, p, nullptr);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(SSM_ERR_WORKSPACE, "gated delta rule: backward workspace of %zu bytes required, %zu given", need,
                workspace_bytes);
  carve_bwd(s, p, align256(workspace));
  fill(p, s, q, k, v, g, beta, scale);
  carve_saved(s, p, align256(const_cast<void*>(saved)));
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
  const cudaError_t e = s.dtype == SSM_BF16 ? run_step<__nv_bfloat16>(s, p, st) : run_step<float>(s, p, st);
  if (e != cudaSuccess) return fail(SSM_ERR_CUDA, "gated delta state update: %s", cudaGetErrorString(e));
  return SSM_OK;
}

}  // extern "C"
