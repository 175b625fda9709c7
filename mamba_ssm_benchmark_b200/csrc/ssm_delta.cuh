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
// The state is kept transposed, S^T (dv x dk), as accumulator fragments: its rows (value channels) are
// independent of one another.  Four warps share a strip of 16 rows: each owns a quarter of dk and two of
// the eight 8-position column tiles of X, U and O.  An accumulator tile is, lane by lane, half of the A
// operand of the next product, so what the warps exchange (the pieces of S, X, U) goes through shared
// memory once, already in operand form.
#pragma once

#include "ssm_common.cuh"
#include "ssm_vec.cuh"

namespace ssm {

constexpr int kC = 64;         // positions per chunk
constexpr int kVec = 5 * kC;   // per-chunk vectors: e^G, e^(G_last - G), beta, G log2(e) as two floats
constexpr int kTri = kC * kC;  // elements of a chunk's T or P

struct Heads {                 // (B, L, H, width), unit stride along the width
  const void* ptr;
  long long sb, sl, sh;
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
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

// Element offset of 8-element column group `grp` of row `row` in a (ROWS x W) bf16 tile.  Its 16-byte groups are
// permuted by the row, so that the eight rows of an ldmatrix hit different banks; a tile of 128 columns is two of 64
// behind one another.  That is the 128-byte swizzle that tcgen05's descriptors name.
template <int W, int ROWS = kC>
__device__ __forceinline__ int tile_off(int row, int grp) {
  static_assert(W == 64 || W == 128, "rows of 128 bytes, or two of these");
  if (W == 128) return (grp >> 3) * (ROWS * 64) + row * 64 + (((grp & 7) ^ (row & 7)) << 3);
  return row * 64 + ((grp ^ (row & 7)) << 3);
}

// B fragments of n tiles j, j + 1 (r[0..1], r[2..3]) and k block kb from a tile stored [n][k].
template <int W, int ROWS = kC>
__device__ __forceinline__ void load_b(uint32_t (&r)[4], uint32_t tile, int j, int kb, int lane) {
  ldsm4(r, tile + 2 * tile_off<W, ROWS>(8 * (j + (lane >> 4)) + (lane & 7), 2 * kb + ((lane >> 3) & 1)));
}
// The same from a tile stored [k][n].
template <int W, int ROWS = kC>
__device__ __forceinline__ void load_bt(uint32_t (&r)[4], uint32_t tile, int j, int kb, int lane) {
  ldsm4t(r, tile + 2 * tile_off<W, ROWS>(16 * kb + (lane & 15), j + (lane >> 4)));
}
// A fragment of the 16 rows from `row` and k block kb from a tile stored [m][k].
template <int W, int ROWS = kC>
__device__ __forceinline__ void load_a(uint32_t (&r)[4], uint32_t tile, int row, int kb, int lane) {
  ldsm4(r, tile + 2 * tile_off<W, ROWS>(row + (lane & 15), 2 * kb + (lane >> 4)));
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

// Tiles j0 .. j0 + 2 NJ - 1 of d += A (NA pieces) x NJ pairs of B fragments of piece pb: the products of pieces
// with MINI <= index sum <= MAXI.  Consecutive instructions go to different accumulators.
// The tensor cores truncate each sum to fp32.  So the small products (index sum >= 1) and the leading ones go to
// accumulators of their own, added at the end: the many truncations of the small ones then count little.
template <int MINI, int MAXI, int NJ, int NA, int NT>
__device__ __forceinline__ void mma_pieces(float (&d)[NT][4], int j0, const uint32_t (&a)[NA][4],
                                           const uint32_t (&b)[NJ][4], int pb) {
#pragma unroll
  for (int i = 0; i < NA; ++i)
    if (i + pb >= MINI && i + pb <= MAXI) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        mma_bf16(d[j0 + 2 * j], a[i], b[j][0], b[j][1]);
        mma_bf16(d[j0 + 2 * j + 1], a[i], b[j][2], b[j][3]);
      }
    }
}
// lead += the leading products, low += the others up to index sum MAXI.
template <int MAXI, int NJ, int NA, int NT>
__device__ __forceinline__ void mma_split(float (&lead)[NT][4], float (&low)[NT][4], int j0, const uint32_t (&a)[NA][4],
                                          const uint32_t (&b)[NJ][4], int pb) {
  mma_pieces<1, MAXI>(low, j0, a, b, pb);
  if (pb == 0) mma_pieces<0, 0>(lead, j0, a, b, 0);
}

template <int NT>
__device__ __forceinline__ void add(float (&c)[NT][4], const float (&x)[NT][4]) {
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) c[j][e] += x[j][e];
}
template <int NT>
__device__ __forceinline__ void zero(float (&c)[NT][4]) {
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) c[j][e] = 0.0f;
}

// ---- strips: kC positions x 16 channels of a (positions, channels) tensor -----------------------------
// Warp w of a strip works on the column tiles w and 7 - w, positions 8 w .. and 56 - 8 w .. (a pair that
// carries the same triangular work for every w).  In the accumulator layout of the transpose element
// (2 r + e) of a tile is position 2 t + e, channel g + 8 r (g = lane / 4, t = lane % 4): a gather of single
// elements from global memory.  So a warp's rows pass through shared memory, 16 bytes at a time, in by
// asynchronous copies a chunk ahead.  The 16-byte units of a row are permuted by the row so that the eight
// rows of a transposing ldmatrix hit different banks.
__device__ __forceinline__ int col_tile(int w, int i) { return i ? 7 - w : w; }

template <typename T>
struct alignas(16) Strip {
  T x[kC * 16];
  static constexpr int kUnit = 16 / (int)sizeof(T);      // elements per unit
  static constexpr int kUnits = 16 / kUnit;              // units per row
  __device__ static int off(int row, int unit) {
    const int s = sizeof(T) == 2 ? (row >> 2) & 1 : (row >> 1) & 3;
    return (row * kUnits + (unit ^ s)) * kUnit;
  }
  __device__ static int row_of(int w, int i) { return 8 * col_tile(w, i >> 3) + (i & 7); }   // i-th of the warp's 16 rows
  // Starts the copy of the warp's rows of `rows` x `cols` elements; the rest becomes zero.
  __device__ void fetch(const T* base, long long sl, int rows, int cols, bool aligned, int w, int lane) {
#pragma unroll
    for (int i = 0; i < kUnits / 2; ++i) {
      const int u = lane + 32 * i, row = row_of(w, u / kUnits), unit = u % kUnits;
      T* dst = x + off(row, unit);
      if (aligned && cols >= 16 && row < rows) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)),
                     "l"(base + row * sl + unit * kUnit)
                     : "memory");
      } else {
#pragma unroll
        for (int e = 0; e < kUnit; ++e)
          dst[e] = row < rows && unit * kUnit + e < cols ? base[row * sl + unit * kUnit + e] : from_f32<T>(0.0f);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  __device__ void arrive() {
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();
  }
  __device__ void read(float (&v)[2][4], int w, int lane) const {
    if constexpr (sizeof(T) == 2) {
      uint32_t r[4];
      ldsm4t(r, smem_u32(x + off(8 * col_tile(w, lane >> 4) + (lane & 7), (lane >> 3) & 1)));
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        v[h >> 1][2 * (h & 1)] = lo_f32(r[h]);
        v[h >> 1][2 * (h & 1) + 1] = hi_f32(r[h]);
      }
    } else {
      const int g = lane >> 2, t = lane & 3;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = 8 * col_tile(w, j) + 2 * t + (e & 1), d = g + 8 * (e >> 1);
          v[j][e] = x[off(c, d >> 2) + (d & 3)];
        }
    }
  }
  __device__ void write(const float (&v)[2][4], int w, int lane) {
    if constexpr (sizeof(T) == 2) {
      const uint32_t a = smem_u32(x + off(8 * col_tile(w, lane >> 4) + (lane & 7), (lane >> 3) & 1));
      asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(a),
                   "r"(pack_bf16(v[0][0], v[0][1])), "r"(pack_bf16(v[0][2], v[0][3])),
                   "r"(pack_bf16(v[1][0], v[1][1])), "r"(pack_bf16(v[1][2], v[1][3]))
                   : "memory");
    } else {
      const int g = lane >> 2, t = lane & 3;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = 8 * col_tile(w, j) + 2 * t + (e & 1), d = g + 8 * (e >> 1);
          x[off(c, d >> 2) + (d & 3)] = v[j][e];
        }
    }
    __syncwarp();
  }
  // Copies the warp's rows out; they may be written again after the next __syncwarp().
  __device__ void flush(T* base, long long sl, int rows, int cols, bool aligned, int w, int lane) const {
#pragma unroll
    for (int i = 0; i < kUnits / 2; ++i) {
      const int u = lane + 32 * i, row = row_of(w, u / kUnits), unit = u % kUnits;
      const T* src = x + off(row, unit);
      if (row >= rows) continue;
      if (aligned && cols >= 16) {
        *reinterpret_cast<uint4*>(base + row * sl + unit * kUnit) = *reinterpret_cast<const uint4*>(src);
      } else {
#pragma unroll
        for (int e = 0; e < kUnit; ++e)
          if (unit * kUnit + e < cols) base[row * sl + unit * kUnit + e] = src[e];
      }
    }
    __syncwarp();
  }
};

// ---- operands exchanged between the warps of a strip: [k block][piece][lane], 16 bytes a lane ------------
// Half h (column tile 2 kb + h) of k block kb's A operand from an accumulator tile.
template <int NP>
__device__ __forceinline__ void put_half(uint4 (*f)[NP][32], int tile, const float (&c)[4], int lane) {
  uint32_t a[NP], b[NP];
  split<NP>(c[0], c[1], a);
  split<NP>(c[2], c[3], b);
#pragma unroll
  for (int i = 0; i < NP; ++i)
    reinterpret_cast<uint2*>(&f[tile >> 1][i][lane])[tile & 1] = make_uint2(a[i], b[i]);
}
__device__ __forceinline__ void get_frag(uint32_t (&a)[4], const uint4& f) {
  a[0] = f.x;
  a[1] = f.y;
  a[2] = f.z;
  a[3] = f.w;
}
// B fragments of the warp's two column tiles from a tile stored [n][k] / [k][n].
template <int W, int ROWS = kC>
__device__ __forceinline__ void load_b2(uint32_t (&r)[4], uint32_t tile, int w, int kb, int lane) {
  ldsm4(r, tile + 2 * tile_off<W, ROWS>(8 * col_tile(w, lane >> 4) + (lane & 7), 2 * kb + ((lane >> 3) & 1)));
}
template <int W, int ROWS = kC>
__device__ __forceinline__ void load_bt2(uint32_t (&r)[4], uint32_t tile, int w, int kb, int lane) {
  ldsm4t(r, tile + 2 * tile_off<W, ROWS>(16 * kb + (lane & 15), col_tile(w, lane >> 4)));
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

// The same as they lie in memory.
template <typename T>
struct alignas(16) Row8 {
  T x[8];
  __device__ __forceinline__ void load(const T* row, int c0, int width, bool vec) {
    if (vec && c0 + 8 <= width) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i)
        reinterpret_cast<uint4*>(x)[i] = reinterpret_cast<const uint4*>(row + c0)[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = c0 + i < width ? row[c0 + i] : from_f32<T>(0.0f);
    }
  }
};

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

// Bulk copy global -> shared, completion on bar; 16-byte aligned, a multiple of 16 bytes.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// What these kernels wait for comes within microseconds.  A poll that runs out takes 3.9 thousand clocks: about a second.
constexpr uint32_t kPolls = 1u << 19;

// A bounded wait; after one that gave up the same thread waits no more, so that the kernel ends (one limit, not one per
// chunk), and starts no copies.
struct Wait {
  int* err;
  bool dead = false;
  __device__ void operator()(uint64_t* bar, uint32_t parity) {
    if (dead) return;
    for (uint32_t it = 0; it < kPolls; ++it)
      if (mbar_try_wait(bar, parity)) return;
    if (err) atomicOr(err, 1);
    dead = true;
  }
  // Before the kernel ends: after a wait that gave up, time for its copies and products in flight to land.
  __device__ void drain() const {
    for (int i = 0; dead && i < 1000; ++i) __nanosleep(1000);
  }
};

// Non-finite values.  A product with a triangular tile multiplies the zeros above its diagonal too, and 0 x inf is NaN: an input
// that is not finite would reach outputs up to 15 positions before it (up to 31 through the blocks of T).  So the products get
// 0 for such values of X and T, a channel's first such position is noted, and at the end of the chunk its outputs from
// there on and its state become NaN: as the recurrence has them, since a state that once is not finite stays so.  A row of
// T with such values, which may come of an overflow as well, makes its X NaN.  Above kBig a float rounds to an infinite bf16
// piece.  On the strips all this is selects and no branch behind X (long prompt 650 us, with branches at the products 683,
// without any of it 655).
constexpr float kBig = 3.3895313e38f;            // the largest bf16
__device__ __forceinline__ float max3_abs(float a, float b, float c) {       // NaN if one of them is
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ bool is_bad(float x) { return !(fabsf(x) <= kBig); }
__device__ __forceinline__ float quiet_nan() { return __int_as_float(0x7fffffff); }

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
  float *pdq, *pdk;            // (B, L, Hv, DKP) per value head, when value heads share key heads
  int* err;
  int B, L, Hk, Hv, dkw, dvw, dvp, n, group;
  float scale;
};

}  // namespace ssm
