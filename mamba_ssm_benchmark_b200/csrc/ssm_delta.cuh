// ssm_delta.cuh — the chunk arithmetic shared by the gated delta rule's kernels.
//
// Per value head, with a state S (dk x dv), G_i the running sum of g inside a chunk of kC positions and
// D_ij = exp(G_i - G_j) for i >= j:
//   A = tril(beta_i D_ij k_i.k_j, -1)     T = (I + A)^-1        P = scale tril(D_ij q_i.k_j)
//   X = beta (V - e^G K S)                U = T X
//   O = scale e^G Q S + P U               S' = e^G_last S + (e^(G_last - G) K)^T U
//
// Products run on mma.sync m16n8k16 with fp32 accumulators.  A float operand is taken as the sum of
// three bf16 pieces (8 bits each, 24 in all), and the products of pieces down to 2^-16 of the largest
// are kept: six for float x float, three for float x bf16, one for bf16 x bf16.  That holds states,
// gradients and their sums to fp32's own rounding, which one bf16 pass (2^-8) does not.
//
// The state is kept transposed, S^T (dv x dk), as accumulator fragments: a warp owns 16 rows (value
// channels).  An accumulator tile pair is, lane by lane, the A operand of the next product, so the
// chain S -> X -> U -> S' of a warp never leaves its registers and needs no barrier.
#pragma once

#include "ssm_common.cuh"

namespace ssm {

constexpr int kC = 64;         // positions per chunk
constexpr int kVec = 5 * kC;   // per-chunk vectors: e^G, e^(G_last - G), beta, G log2(e) as two floats
constexpr int kTri = kC * kC;  // elements of a chunk's T or P

struct Heads {                 // (B, L, H, width), unit stride along the width
  const void* ptr;
  long long sb, sl, sh;
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// lo in the low half
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float lo_f32(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float hi_f32(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }

// x0, x1 as the sums of NP bf16 pieces each, the largest first.
template <int NP>
__device__ __forceinline__ void split(float x0, float x1, uint32_t (&p)[NP]) {
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    p[i] = pack_bf16(x0, x1);
    if (i + 1 < NP) {
      x0 -= lo_f32(p[i]);
      x1 -= hi_f32(p[i]);
    }
  }
}

// Element offset of 8-element column group `grp` of row `row` in a (rows x W) bf16 tile whose 16-byte
// groups are permuted by the row, so that the eight rows of an ldmatrix hit different banks.
template <int W>
__device__ __forceinline__ int tile_off(int row, int grp) {
  return row * W + ((grp ^ (row & 7)) << 3);
}

// B fragments of n tiles j, j + 1 (r[0..1], r[2..3]) and k block kb from a tile stored [n][k].
template <int W>
__device__ __forceinline__ void load_b(uint32_t (&r)[4], uint32_t tile, int j, int kb, int lane) {
  ldsm4(r, tile + 2 * tile_off<W>(8 * (j + (lane >> 4)) + (lane & 7), 2 * kb + ((lane >> 3) & 1)));
}
// The same from a tile stored [k][n].
template <int W>
__device__ __forceinline__ void load_bt(uint32_t (&r)[4], uint32_t tile, int j, int kb, int lane) {
  ldsm4t(r, tile + 2 * tile_off<W>(16 * kb + (lane & 15), j + (lane >> 4)));
}
// A fragment of the 16 rows from `row` and k block kb from a tile stored [m][k].
template <int W>
__device__ __forceinline__ void load_a(uint32_t (&r)[4], uint32_t tile, int row, int kb, int lane) {
  ldsm4(r, tile + 2 * tile_off<W>(row + (lane & 15), 2 * kb + (lane >> 4)));
}

// The A operand of k block kb from accumulator tiles 2 kb, 2 kb + 1, in NP pieces.
template <int NP, int NT>
__device__ __forceinline__ void acc_to_a(const float (&c)[NT][4], int kb, uint32_t (&a)[NP][4]) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      uint32_t p[NP];
      split<NP>(c[2 * kb + h][2 * r], c[2 * kb + h][2 * r + 1], p);
#pragma unroll
      for (int i = 0; i < NP; ++i) a[i][2 * h + r] = p[i];
    }
}

// d0, d1 += A (NA pieces) x the B fragments of piece pb, every product of pieces with index sum <= MAXI.
template <int NA, int MAXI>
__device__ __forceinline__ void mma_pieces(float (&d0)[4], float (&d1)[4], const uint32_t (&a)[NA][4],
                                           const uint32_t (&b)[4], int pb) {
#pragma unroll
  for (int i = 0; i < NA; ++i)
    if (i + pb <= MAXI) {
      mma_bf16(d0, a[i], b[0], b[1]);
      mma_bf16(d1, a[i], b[2], b[3]);
    }
}

template <int NT>
__device__ __forceinline__ void zero(float (&c)[NT][4]) {
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) c[j][e] = 0.0f;
}

// (positions x value channels) of a head read in the accumulator layout of its transpose: element
// (2 r + e) of tile j is position 8 j + 2 t + e, channel g + 8 r (g = lane / 4, t = lane % 4).
template <typename T>
__device__ __forceinline__ void load_vt(const T* base, long long sl, int rows, int cols, int lane, float (&v)[kC / 8][4]) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int j = 0; j < kC / 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = 8 * j + 2 * t + (e & 1), d = g + 8 * (e >> 1);
      v[j][e] = c < rows && d < cols ? to_f32(base[(long long)c * sl + d]) : 0.0f;
    }
}
template <typename T>
__device__ __forceinline__ void store_vt(T* base, long long sl, int rows, int cols, int lane, const float (&v)[kC / 8][4]) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int j = 0; j < kC / 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = 8 * j + 2 * t + (e & 1), d = g + 8 * (e >> 1);
      if (c < rows && d < cols) base[(long long)c * sl + d] = from_f32<T>(v[j][e]);
    }
}
// 16 rows of a dense fp32 [channel][W] tile from / to accumulators.
template <int NT>
__device__ __forceinline__ void store_acc(float* base, int W, int lane, const float (&c)[NT][4]) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    *reinterpret_cast<float2*>(base + (size_t)g * W + 8 * j + 2 * t) = make_float2(c[j][0], c[j][1]);
    *reinterpret_cast<float2*>(base + (size_t)(g + 8) * W + 8 * j + 2 * t) = make_float2(c[j][2], c[j][3]);
  }
}

// Bulk copy global -> shared, completion on bar; 16-byte aligned, a multiple of 16 bytes.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

struct DeltaParams {
  Heads q, k, v, o;            // o: the forward's output / the backward's incoming gradient of it
  Heads dq, dk, dv;
  const float *g, *beta;       // (B, L, Hv), unit stride along the heads
  long long gsb, gsl, bsb, bsl;
  float *dg, *dbeta;           // (B, L, Hv) dense
  const float* h0;             // (B, Hv, dk, dv) or null; the backward reads the last state's gradient here
  float* last;                 // (B, Hv, dk, dv) or null; the backward writes the first state's gradient here
  // workspace
  __nv_bfloat16 *kimg, *qimg;  // (B, Hk, n, pieces, kC, DKP)
  __nv_bfloat16 *timg, *pimg;  // (B, Hv, n, 3, kC, kC)
  float* vec;                  // (B, Hv, n, kVec)
  float* states;               // (B, Hv, n, dvp, DKP): S^T entering the chunk
  float* us;                   // (B, Hv, n, dvp, kC): U^T
  float* dstates;              // the gradient of the state leaving the chunk, like states
  float* dxs;                  // dX^T, like us
  float *pdq, *pdk;            // (B, L, Hv, dk) per value head, when value heads share key heads
  int* err;
  int B, L, Hk, Hv, dkw, dvw, dvp, n, group;
  float scale;
};

}  // namespace ssm
