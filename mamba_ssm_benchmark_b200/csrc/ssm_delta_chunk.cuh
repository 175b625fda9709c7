// ssm_delta_chunk.cuh — the gated delta rule's backward, all chunks at once, on tcgen05.  With
//   E1 = dO S^T,  E2 = dX S^T,  E3 = U dS'^T,  N = -tril(D dX U^T, -1),  M = scale tril(D dO U^T, -1),
//   m_i = scale dO_i.U_i (the diagonal, where D = 1 has no gradient)
//   H = N K - e^G E2                         (the gradient of beta k)
//   dQ = scale e^G E1 + M K,   dK = beta H + C,  C = N^T (beta K) + M^T Q + e^(G_last - G) E3
//   dbeta_i = dX_i.V_i + k_i.H_i
//   dG_i = q_i.dQ_i + beta_i k_i.H_i - k_i.C_i;  the last position also gets
//          sum_i e^(G_last - G_i) k_i.E3_i + e^G_last <S, dS'>
// after which dQ_i gets m_i k_i and dK_i gets m_i q_i; dg is dG summed from the end of the chunk.  Every
// exponent's gradient is thus a row product of gradients that are formed anyway; k.k and q.k are not needed again.
//
// One CTA per SM walks over (chunk, head, batch).  dv is walked 16 channels at a time: bulk copies bring slabs of S,
// dS', U and dX (fp32) ahead; sixteen warps split them into bf16 pieces in 128-byte-swizzled tiles, two slabs' worth,
// one warp multiplies them, and one copies and does the last sums along a chunk.  The 128 rows of a product are two
// operands of 64 positions on top of one another: [dO; dX] [S | U]^T, [0; U] dS'^T, then [M; N] K and
// [0; (beta N)^T] K + [0; M^T] Q; so a thread meets H and C of one position, or dQ.  Sums of small products and of
// leading ones are kept apart where tensor memory has the columns for it (E3 at dk > 64 has not).
//
// 5120 chunks of 128 x 128 (bf16): 584 us, on mma.sync 1020.  Of 29 thousand clocks a chunk the slabs take 16, where
// pieces written and operands read fill shared memory's bandwidth; the 13 behind the last slab are overlapped by
// nothing, as the accumulators fill tensor memory.
#pragma once

#include "ssm_delta_tc.cuh"

namespace ssm {

constexpr int kSL = 16;                          // channels of a slab: one k block

template <int DKP>
struct alignas(128) ChunkSlab {                  // as it lies in global memory
  float S[kSL * DKP], dS[kSL * DKP], U[kSL * kC], dX[kSL * kC];
};
template <int NP, int DKP>
struct alignas(1024) ChunkPieces {               // tiles [channel][position or dk]; SU: S and beside it U
  __nv_bfloat16 dO[NP][kSL * kC], dX[3][kSL * kC], SU[3][kSL * (DKP + kC)], dS[3][kSL * DKP];
};
struct alignas(1024) ChunkTri {
  __nv_bfloat16 MN[3][2][kTri], Nb[3][kTri];     // Nb: rows of N times beta
};
template <int NP, int DKP>
struct alignas(1024) ChunkSmem {
  static constexpr int RB = NP == 3 && DKP == 128 ? 1 : 4;      // slabs on their way
  __nv_bfloat16 zero[kSL * kC];                  // lowest: the distance to every other tile is positive
  union {
    ChunkPieces<NP, DKP> x[2];
    ChunkTri tri;                                // after the last slab
    float4 rows[16][32 * 8];                     // after the last product: per warp, see tc_store_rows
  };
  __nv_bfloat16 k[NP][kC * DKP], q[NP][kC * DKP];
  ChunkSlab<DKP> slab[RB];
  alignas(16) float vec[kVec];
  float dots[4][4][kC];                          // q.dQ, k.H, k.C, e^(G_last - G) k.E3; by quarter of dk
  float dxv[2][kC];                              // dX.V by half of a slab
  float sds[16];                                 // <S, dS'> by warp
  float m[kC];                                   // the diagonal of M
  uint64_t full_slab[RB], free_slab[RB], full_tiles, ready[2], done[2], ready_tri, done_tri, free_tiles;
  uint32_t tmem;
};
constexpr int kChunkThreads = 512 + 64;

// Columns of tensor memory: E3; then [E1; E2] and beside it [dO; dX] U^T, small sums and, kLead further, leading ones.
// [M; N] K and what makes C take the latter's place.  With kStacked the pieces of K (or Q) are one wide operand and
// their products lie kStacked columns apart, by index sum: half the instructions (1024 chunks, fp32, dk 64: 113 -> 102 us).
template <int NP, int DKP>
struct ChunkCols {
  static constexpr int kStacked = NP == 3 && DKP == 64 ? 64 : 0;
  enum : uint32_t { kE3 = 0, kE3Lead = 64, kE = 128, kU = kE + DKP, kLead = DKP + kC, kMNK = 128 };
  static constexpr uint32_t kCC = kMNK + (kStacked ? 3 * kStacked : DKP);
  static_assert(kE + 2 * kLead <= kTcCols && kCC + (kStacked ? 3 * kStacked : DKP) <= kTcCols, "tensor memory");
};

__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t high, uint32_t idesc, bool accumulate,
                                          uint32_t issue) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(high), "r"(idesc), "r"((uint32_t)accumulate), "r"(issue)
      : "memory");
}
constexpr uint32_t kTcAcrossA = 1u << 15;        // A read across its rows, [k][m]
// The low descriptor word of two 64-row blocks of A, the upper one at `low`.
__device__ __forceinline__ uint32_t tc_pair(uint32_t low, uint32_t high) { return tc_desc(low, high - low); }

// Two or four neighbours in three pieces, `stride` apart.
template <int N>
__device__ __forceinline__ void put_values(const float (&v)[N], __nv_bfloat16* o, int stride) {
  uint32_t q[N / 2][3];
#pragma unroll
  for (int e = 0; e < N / 2; ++e) split<3>(v[2 * e], v[2 * e + 1], q[e]);
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    if constexpr (N == 4) *reinterpret_cast<uint2*>(o + k * stride) = make_uint2(q[0][k], q[1][k]);
    else *reinterpret_cast<uint32_t*>(o + k * stride) = q[0][k];
  }
}

template <typename T, int NP, int DKP>
__global__ void __launch_bounds__(kChunkThreads, 1) delta_bwd_chunk(const __grid_constant__ DeltaParams p) {
  using Smem = ChunkSmem<NP, DKP>;
  using Cols = ChunkCols<NP, DKP>;
  constexpr int RB = Smem::RB, QK = DKP / 4;
  constexpr bool kApart = DKP == 64;             // E3's small sums have columns of their own
  Smem& s = tc_smem<Smem>();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int items = p.n * p.Hv * p.B, slabs = p.dvp / kSL;           // (chunk, head, batch); slabs of each
  if (tid == 0) {
    for (int i = 0; i < RB; ++i) {
      mbar_init(&s.full_slab[i], 1);
      mbar_init(&s.free_slab[i], 16);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.ready[i], 16);
      mbar_init(&s.done[i], 1);
    }
    mbar_init(&s.full_tiles, 1);
    mbar_init(&s.ready_tri, 16);
    mbar_init(&s.done_tri, 1);
    mbar_init(&s.free_tiles, 17);
    fence_mbar_init();
  }
  if (warp == 16) tc_alloc(&s.tmem, kTcCols);
  for (int i = tid; i < kSL * kC / 8; i += kChunkThreads) reinterpret_cast<uint4*>(s.zero)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = __shfl_sync(0xffffffffu, s.tmem, 0);
  Wait wait{p.err};

  if (warp == 17) {
    // ---- copies; dbeta and dg ----
    auto fetch_slab = [&](int it) {              // slab number `it` of this CTA, counted over its items
      const size_t at = blockIdx.x + (size_t)(it / slabs) * gridDim.x;
      if (lane != 0 || wait.dead || at >= (size_t)items) return;
      const size_t row = at * p.dvp + it % slabs * kSL;
      auto& d = s.slab[it % RB];
      uint64_t* bar = &s.full_slab[it % RB];
      mbar_arrive_expect_tx(bar, sizeof(d.S) + sizeof(d.dS) + sizeof(d.U) + sizeof(d.dX));
      bulk_load(d.S, p.states + row * DKP, sizeof(d.S), bar);
      bulk_load(d.dS, p.dstates + row * DKP, sizeof(d.dS), bar);
      bulk_load(d.U, p.us + row * kC, sizeof(d.U), bar);
      bulk_load(d.dX, p.dxs + row * kC, sizeof(d.dX), bar);
    };
    auto fetch_tiles = [&](int item) {
      if (lane != 0 || wait.dead || item >= items) return;
      const int h = item / p.n % p.Hv, b = item / p.n / p.Hv;
      const size_t atk = ((size_t)b * p.Hk + h / p.group) * p.n + item % p.n;
      mbar_arrive_expect_tx(&s.full_tiles, sizeof(s.k) + sizeof(s.q) + sizeof(s.vec));
      bulk_load(s.k, p.kimg + atk * (NP * kC * DKP), sizeof(s.k), &s.full_tiles);
      bulk_load(s.q, p.qimg + atk * (NP * kC * DKP), sizeof(s.q), &s.full_tiles);
      bulk_load(s.vec, p.vec + (size_t)item * kVec, sizeof(s.vec), &s.full_tiles);
    };
    for (int i = 0; i < RB; ++i) fetch_slab(i);
    fetch_tiles(blockIdx.x);
    int it = 0;
#pragma unroll 1
    for (int item = blockIdx.x, turn = 0; item < items; item += gridDim.x, ++turn) {
      const int ch = item % p.n, h = item / p.n % p.Hv, b = item / p.n / p.Hv, rows = min(kC, p.L - ch * kC);
      const long long t0 = (long long)ch * kC;
      for (int j = 0; j < slabs; ++j, ++it) {
        wait(&s.free_slab[it % RB], (it / RB) & 1);
        __syncwarp();
        fetch_slab(it + RB);
      }
      wait(&s.full_tiles, turn & 1);
      asm volatile("bar.sync 2, 544;" ::: "memory");       // the dots are there
      const float* vec = s.vec;
      float dG[2], tail = 0.0f;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 2 * lane + e;
        auto sum = [&](int w) { return (s.dots[w][0][r] + s.dots[w][1][r]) + (s.dots[w][2][r] + s.dots[w][3][r]); };
        const float kH = sum(1);
        dG[e] = sum(0) + vec[2 * kC + r] * kH - sum(2);
        tail += sum(3);
        if (r < rows) p.dbeta[((size_t)b * p.L + t0 + r) * p.Hv + h] = (s.dxv[0][r] + s.dxv[1][r]) + kH;
      }
      tail = group_allreduce<32, 1>(tail);
      float sds = 0.0f;
#pragma unroll
      for (int e = 0; e < 16; ++e) sds += s.sds[e];
      tail = fmaf(vec[kC - 1], sds, tail);
      float run = dG[0] + dG[1];
#pragma unroll
      for (int k = 1; k < 32; k <<= 1) {
        const float down = __shfl_down_sync(0xffffffffu, run, k);
        if (lane + k < 32) run += down;
      }
      run += tail;
      if (2 * lane < rows) p.dg[((size_t)b * p.L + t0 + 2 * lane) * p.Hv + h] = run;
      if (2 * lane + 1 < rows) p.dg[((size_t)b * p.L + t0 + 2 * lane + 1) * p.Hv + h] = run - dG[0];
      __syncwarp();
      if (lane == 0) tc_arrive(&s.free_tiles);
      wait(&s.free_tiles, turn & 1);             // so the others do not write these sums again before they are read
      fetch_tiles(item + gridDim.x);
    }
    __syncwarp();
  } else if (warp == 16) {
    // ---- products ----
    const uint32_t issue = lane == 0, zero = smem_u32(s.zero);
    int it = 0;
    for (int item = blockIdx.x, turn = 0; item < items; item += gridDim.x, ++turn) {
      for (int j = 0; j < slabs; ++j, ++it) {
        auto& x = s.x[it & 1];
        wait(&s.ready[it & 1], (it >> 1) & 1);
        tc_fence_after();
        const uint32_t tSU = smem_u32(x.SU), tdS = smem_u32(x.dS), tX = smem_u32(x.dX), tO = smem_u32(x.dO);
        constexpr uint32_t kOne = kSL * kC * 2, kRow = kSL * DKP * 2;           // bytes of a tile's piece
        const bool more = j > 0;
        bool any = more, any3 = more;
#pragma unroll
        for (int lead = 0; lead < 2; ++lead)     // small products first: E3's share its columns at dk > 64
#pragma unroll
          for (int a = 0; a < 3; ++a)
#pragma unroll
            for (int b = 0; b < 3; ++b) {
              if (a + b > 2 || (a + b == 0) != (lead == 1)) continue;
              const uint32_t ox = tc_pair(a < NP ? tO + a * kOne : zero, tX + a * kOne);
              const uint32_t zu = tc_pair(zero, tSU + a * (kRow + kOne) + kRow);
              const uint32_t bSU = tc_desc(tSU + b * (kRow + kOne), kOne), bdS = tc_desc(tdS + b * kRow, kOne);
              tc_mma_ss(tm + Cols::kE + (lead ? Cols::kLead : 0), ox, bSU, kTcDescHigh, tc_idesc<true>(DKP + kC) | kTcAcrossA,
                        lead ? more : any, issue);
              tc_mma_ss(tm + (kApart && lead ? Cols::kE3Lead : Cols::kE3), zu, bdS, kTcDescHigh, tc_idesc<true>(DKP) | kTcAcrossA,
                        kApart && lead ? more : any3, issue);
              any = any3 = true;
            }
        if (issue) tc_commit(&s.done[it & 1]);
      }
      wait(&s.full_tiles, turn & 1);
      wait(&s.ready_tri, turn & 1);
      tc_fence_after();
      const uint32_t tMN = smem_u32(s.tri.MN), tNb = smem_u32(s.tri.Nb), sk = smem_u32(s.k), sq = smem_u32(s.q);
      constexpr uint32_t kTile = kTri * 2, kKey = kC * DKP * 2;
      const uint32_t kAcrossA = tc_idesc<true>(DKP) | kTcAcrossA;
      if constexpr (Cols::kStacked != 0) {
#pragma unroll
        for (int a = 0; a < 3; ++a)              // pieces 0 .. 2 - a of K and Q
#pragma unroll
          for (int st = 0; st < kC / 16; ++st) {
            constexpr uint32_t kBlock = kC * 64 * 2;
            const uint32_t bk = tc_desc(sk + st * 2048, kBlock), bq = tc_desc(sq + st * 2048, kBlock);
            const uint32_t idesc = tc_idesc<true>((3 - a) * DKP), to = a * Cols::kStacked;
            const bool more = a + st > 0;
            tc_mma_ss(tm + Cols::kMNK + to, tc_desc(tMN + 2 * a * kTile + st * 32, 16), bk, kTcDescHigh, idesc, more, issue);
            tc_mma_ss(tm + Cols::kCC + to, tc_pair(zero, tNb + a * kTile + st * 2048), bk, kTcDescHigh, idesc | kTcAcrossA, more,
                      issue);
            tc_mma_ss(tm + Cols::kCC + to, tc_pair(zero, tMN + 2 * a * kTile + st * 2048), bq, kTcDescHigh, idesc | kTcAcrossA,
                      true, issue);
          }
      } else {
        bool more = false;
#pragma unroll
        for (int lead = 0; lead < 2; ++lead)
#pragma unroll
          for (int a = 0; a < 3; ++a)
#pragma unroll
            for (int b = 0; b < NP; ++b) {
              if (a + b > 2 || (a + b == 0) != (lead == 1)) continue;
#pragma unroll
              for (int st = 0; st < kC / 16; ++st) {
                const uint32_t at = b * kKey + st * 2048;
                const uint32_t bk = tc_desc(sk + at, kC * 64 * 2), bq = tc_desc(sq + at, kC * 64 * 2);
                tc_mma_ss(tm + Cols::kMNK, tc_desc(tMN + 2 * a * kTile + st * 32, 16), bk, kTcDescHigh, tc_idesc<true>(DKP), more,
                          issue);
                tc_mma_ss(tm + Cols::kCC, tc_pair(zero, tNb + a * kTile + st * 2048), bk, kTcDescHigh, kAcrossA, more, issue);
                tc_mma_ss(tm + Cols::kCC, tc_pair(zero, tMN + 2 * a * kTile + st * 2048), bq, kTcDescHigh, kAcrossA, true, issue);
                more = true;
              }
            }
      }
      if (issue) tc_commit(&s.done_tri);
    }
    __syncwarp();
  } else {
    // ---- splitting, and what follows the products ----
    const uint32_t my = tm + ((uint32_t)(32 * (warp & 3)) << 16);
    const int quarter = warp >> 2, row = 32 * (warp & 3) + lane, i = row & 63;      // row of the products, position
    const bool upper = (warp & 3) >= 2;                                          // dX, U, N: dK; else dO, M: dQ
    // beside its part of S and dS', a thread splits 8 values of U, dX or dO, or adds to dX.V, by `role`
    const int role = tid >> 7, lc = tid & 63, lg = (tid >> 6) & 1;                // of dO or V: position, half of a slab
    const T* gbase = static_cast<const T*>(role == 2 ? p.o.ptr : p.v.ptr);
    const long long gsb = role == 2 ? p.o.sb : p.v.sb, gsl = role == 2 ? p.o.sl : p.v.sl, gsh = role == 2 ? p.o.sh : p.v.sh;
    const bool gvec = role == 2 ? rows_aligned16(p.o, sizeof(T)) : rows_aligned16(p.v, sizeof(T));
    int it = 0;
#pragma unroll 1
    for (int item = blockIdx.x, turn = 0; item < items; item += gridDim.x, ++turn) {
      const int ch = item % p.n, h = item / p.n % p.Hv, b = item / p.n / p.Hv, hk = h / p.group;
      const int rows = min(kC, p.L - ch * kC);
      const long long t0 = (long long)ch * kC;
      const T* rowp = gbase + b * gsb + (t0 + lc) * gsl + h * gsh;
      const int width = lc < rows ? p.dvw : 0;
      Row8<T> ahead;
      if (role >= 2) ahead.load(rowp, 8 * lg, width, gvec);
      float dot = 0.0f, dxv = 0.0f;
      for (int j = 0; j < slabs; ++j, ++it) {
        auto& x = s.x[it & 1];
        const auto& raw = s.slab[it % RB];
        wait(&s.full_slab[it % RB], (it / RB) & 1);
        if (j >= 2) wait(&s.done[it & 1], ((it >> 1) - 1) & 1);       // (earlier items' products are long done)
        {
          constexpr int kN = kSL * DKP / 512;      // values of S and of dS': 4 or 2
          const int r = tid * kN / DKP, col = tid * kN % DKP, in8 = (tid & (8 / kN - 1)) * kN;
          float a[kN], c[kN];
          vec_load<float, kN>(raw.S + tid * kN, a);
          vec_load<float, kN>(raw.dS + tid * kN, c);
#pragma unroll
          for (int e = 0; e < kN; ++e) dot = fmaf(a[e], c[e], dot);
          const int off = tile_off<DKP, kSL>(r, col >> 3) + in8;
          put_values(a, x.SU[0] + off, kSL * (DKP + kC));
          put_values(c, x.dS[0] + off, kSL * DKP);
        }
        if (role < 2) {
          const float* src = role ? raw.dX : raw.U;
          __nv_bfloat16* dst = role ? x.dX[0] : x.SU[0] + kSL * DKP;
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const int at = (tid & 127) + 128 * q, r = at / (kC / 4), grp = at % (kC / 4);
            float a[4];
            load4(src + 4 * at, a);
            put_values(a, dst + tile_off<kC, kSL>(r, grp >> 1) + 4 * (grp & 1), role ? kSL * kC : kSL * (DKP + kC));
          }
        } else {
          if (role == 2) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              uint32_t q[NP];
              split<NP>(to_f32(ahead.x[e]), 0.0f, q);
#pragma unroll
              for (int k = 0; k < NP; ++k)
                x.dO[k][tile_off<kC, kSL>(8 * lg + e, lc >> 3) + (lc & 7)] = __ushort_as_bfloat16((unsigned short)(q[k] & 0xffff));
            }
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) dxv = fmaf(raw.dX[(8 * lg + e) * kC + lc], to_f32(ahead.x[e]), dxv);
          }
          if (j + 1 < slabs) ahead.load(rowp, (j + 1) * kSL + 8 * lg, width, gvec);
        }
        fence_proxy_async_smem();
        tc_ready(&s.ready[it & 1]);
        if (lane == 0) tc_arrive(&s.free_slab[it % RB]);
      }
      dot = group_allreduce<32, 1>(dot);
      wait(&s.full_tiles, turn & 1);
      if (slabs > 1) wait(&s.done[(it - 2) & 1], ((it - 2) >> 1) & 1);
      wait(&s.done[(it - 1) & 1], ((it - 1) >> 1) & 1);
      tc_fence_after();
      if (role == 3) s.dxv[lg][lc] = dxv;
      if (lane == 0) s.sds[warp] = dot;
      const float* vec = s.vec;
      const float eg = vec[i], la = vec[kC + i], be = vec[2 * kC + i];
      float E[QK];                                 // this row of [E1; E2], scaled; then of dQ or dK
      {
        // M or N, 16 columns of a row, into the tiles where the slabs were; and beta N
        float x[16], y[16];
        const int c0 = 16 * quarter;
        tc_load_f32(my + Cols::kU + c0, x);
        tc_load_f32(my + Cols::kU + Cols::kLead + c0, y);
        const float gh = vec[3 * kC + i], gl = vec[4 * kC + i], f = upper ? -1.0f : p.scale;
#pragma unroll
        for (int e0 = 0; e0 < 16; e0 += 4) {
          float h4[4], l4[4];
          load4(vec + 3 * kC + c0 + e0, h4);
          load4(vec + 4 * kC + c0 + e0, l4);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int e = e0 + q, c = c0 + e;
            x[e] += y[e];
            if (!upper && c == i) s.m[i] = p.scale * x[e];
            x[e] = i > c ? f * ex2((gh - h4[q]) + (gl - l4[q])) * x[e] : 0.0f;
          }
        }
#pragma unroll
        for (int g8 = 0; g8 < 2; ++g8) {
          float v[8], w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            v[e] = x[8 * g8 + e];
            w[e] = be * v[e];
          }
          const int off = tile_off<kC>(i, (c0 >> 3) + g8);
          put_pieces<3>(v, s.tri.MN[0][upper], nullptr, off, 2 * kTri);
          if (upper) put_pieces<3>(w, s.tri.Nb[0], nullptr, off, kTri);
        }
        const float e1 = upper ? -eg : p.scale * eg;
#pragma unroll
        for (int j = 0; j < QK / 16; ++j) {
          tc_load_f32(my + Cols::kE + quarter * QK + 16 * j, x);
          tc_load_f32(my + Cols::kE + Cols::kLead + quarter * QK + 16 * j, y);
#pragma unroll
          for (int e = 0; e < 16; ++e) E[16 * j + e] = e1 * (x[e] + y[e]);
        }
      }
      fence_proxy_async_smem();
      tc_ready(&s.ready_tri);
      asm volatile("bar.sync 1, 512;" ::: "memory");       // m is there
      wait(&s.done_tri, turn & 1);
      tc_fence_after();
      auto load_sums = [&](uint32_t at, float (&v)[16]) {
        tc_load_f32(my + at, v);
        if constexpr (Cols::kStacked != 0) {
          float a[16], b[16];
          tc_load_f32(my + at + Cols::kStacked, a);
          tc_load_f32(my + at + 2 * Cols::kStacked, b);
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] += a[e] + b[e];
        }
      };
      float qd = 0.0f, kh = 0.0f, kc = 0.0f, ke = 0.0f;
      const float m = s.m[i];
      auto row_of = [&](const __nv_bfloat16* tile, int col, float (&v)[16]) {       // of K or Q, 16 columns, whole
#pragma unroll
        for (int g8 = 0; g8 < 2; ++g8) {
          float t[8];
          vec_load<__nv_bfloat16, 8>(tile + tile_off<DKP>(i, (col >> 3) + g8), t);
#pragma unroll
          for (int n = 1; n < NP; ++n) {
            float u[8];
            vec_load<__nv_bfloat16, 8>(tile + n * (kC * DKP) + tile_off<DKP>(i, (col >> 3) + g8), u);
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] += u[e];
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) v[8 * g8 + e] = t[e];
        }
      };
#pragma unroll
      for (int j = 0; j < QK / 16; ++j) {
        const int col = quarter * QK + 16 * j;
        float* o = E + 16 * j;
        float y[16], z[16], v[16];
        load_sums(Cols::kMNK + col, y);
#pragma unroll
        for (int e = 0; e < 16; ++e) o[e] += y[e];
        if (upper) {
          row_of(s.k[0], col, v);
          tc_load_f32(my + Cols::kE3 + col, y);
          if (kApart) {
            tc_load_f32(my + Cols::kE3Lead + col, z);
#pragma unroll
            for (int e = 0; e < 16; ++e) y[e] += z[e];
          }
          load_sums(Cols::kCC + col, z);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            y[e] *= la;
            kh = fmaf(v[e], o[e], kh);
            ke = fmaf(v[e], y[e], ke);
            y[e] += z[e];
            kc = fmaf(v[e], y[e], kc);
          }
          row_of(s.q[0], col, v);
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = fmaf(m, v[e], fmaf(be, o[e], y[e]));
        } else {
          row_of(s.q[0], col, v);
#pragma unroll
          for (int e = 0; e < 16; ++e) qd = fmaf(v[e], o[e], qd);
          row_of(s.k[0], col, v);
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = fmaf(m, v[e], o[e]);
        }
      }
      const int first = i - lane, col = quarter * QK;              // the warp's first position and column
      if (p.group > 1) {           // per value head, summed by delta_sum_heads
        float* o = (upper ? p.pdk : p.pdq) + (((size_t)b * p.L + t0 + first) * p.Hv + h) * DKP + col;
        tc_store_rows<QK / 4>(s.rows[warp], o, p.Hv * DKP, rows - first, E, lane);
      } else if (i < rows) {
        const Heads& out = upper ? p.dk : p.dq;
        T* o = static_cast<T*>(const_cast<void*>(out.ptr)) + b * out.sb + (t0 + i) * out.sl + hk * out.sh + col;
        if (col + QK <= p.dkw && (reinterpret_cast<uintptr_t>(o) & 15) == 0) {
          constexpr int kN = 16 / (int)sizeof(T);
#pragma unroll
          for (int e = 0; e < QK; e += kN) {
            float t[kN];
#pragma unroll
            for (int u = 0; u < kN; ++u) t[u] = E[e + u];
            vec_store<T, kN>(o + e, t);
          }
        } else {
#pragma unroll
          for (int e = 0; e < QK; ++e)
            if (col + e < p.dkw) o[e] = from_f32<T>(E[e]);
        }
      }
      __syncwarp();
      if (upper) {
        s.dots[1][quarter][i] = kh;
        s.dots[2][quarter][i] = kc;
        s.dots[3][quarter][i] = ke;
      } else {
        s.dots[0][quarter][i] = qd;
      }
      asm volatile("bar.sync 2, 544;" ::: "memory");       // the dots are there; nothing is read of rows any more
      tc_fence_before();
      if (lane == 0) tc_arrive(&s.free_tiles);
    }
    tc_fence_before();
  }
  wait.drain();
  __syncthreads();
  if (warp == 16) tc_free(tm, kTcCols);
}

}  // namespace ssm
