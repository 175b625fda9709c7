// ssm_delta_tc.cuh — the gated delta rule's chains on the fifth-generation tensor cores.
//
// The strips of ssm_delta.cu cut a chunk's chain finely, which wins while they do not fill the GPU.  With more
// heads the tensor pipe decides, and mma.sync has a quarter of its rate.  Here one CTA carries 128 value
// channels of a head (the M of tcgen05.mma): S^T lies across 512 threads, a thread holding one channel and a
// quarter of dk in registers.  Each product takes its left operand (pieces of S, X, U: three bf16 each) from tensor
// memory, where the threads put it, and its right one from shared memory, where a bulk copy put the tile; the
// accumulators are read back, combined and split for the next product.  Small products of pieces come before the
// leading ones in every sum, so that the accumulators' truncations count only at the end.
//
// A chunk is three dependent rounds of products with a register pass after each; a warp of its own issues them:
//   forward   S -> [K S, Q S] -> X -> [T X] -> U -> [P U, K^T U]
//   backward  dS' -> [K dS', P^T dO] -> Y -> [T^T Y] -> dX -> [Q^T dO, K^T dX]
//
// 80 heads of 128 x 128, 4096 positions, bf16, training: 439 us forward (14 thousand clocks a chunk) and 463 us
// backward; the strips take 856 and 1146, and with half the threads these kernels 456 and 562 (fp32, dk 64: 67 and 77
// instead of 60 and 63).  The rounds' products take 2.4, 1.7 and 1.8 thousand clocks, about 53 an instruction whatever
// its N up to 64; the register passes and the saved states' stores take the rest.
#pragma once

#include "ssm_delta.cuh"

namespace ssm {

// ---- tensor memory and tcgen05 --------------------------------------------------------------
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_alloc(uint32_t* slot, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tc_free(uint32_t base, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols));
}
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
// D (128 x N, fp32) (+)= A (128 x 16 bf16, tensor memory) x B (16 x N bf16, shared memory), issued by the lane whose
// `issue` is set.  The whole warp calls it with the same operands, which thus stay in uniform registers: from a
// branch that one lane takes, each instruction cost 53 clocks to issue.
__device__ __forceinline__ void tc_mma(uint32_t d, uint32_t a, uint32_t b, uint32_t b_high, uint32_t idesc,
                                       bool accumulate, uint32_t issue) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(b_high), "r"(idesc), "r"((uint32_t)accumulate), "r"(issue)
      : "memory");
}
__device__ __forceinline__ void tc_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_store8(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// 16 columns of this warp's 32 lanes
__device__ __forceinline__ void tc_load_f32(uint32_t addr, float (&v)[16]) {
  uint32_t r[16];
  __syncwarp();
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
  tc_wait_load();
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
// 16 values as NP pieces of 8 packed columns each, `stride` columns apart
template <int NP>
__device__ __forceinline__ void tc_put(uint32_t addr, int stride, const float (&v)[16]) {
  __syncwarp();
  uint32_t r[NP][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint32_t x[NP];
    split<NP>(v[2 * i], v[2 * i + 1], x);
#pragma unroll
    for (int k = 0; k < NP; ++k) r[k][i] = x[k];
  }
#pragma unroll
  for (int k = 0; k < NP; ++k) tc_store8(addr + k * stride, r[k]);
}

// Shared memory descriptors of the 128-byte-swizzled tiles (rows of 64 bf16): read along the rows, [n][k] (stride
// 1024 bytes between groups of eight rows), or across them, [k][n] (the same, and 8192 bytes from one block of 64
// columns to the next).  The low word is the address and that distance, the high word is the same for all.
__device__ __forceinline__ uint32_t tc_desc(uint32_t addr, uint32_t lead_bytes) {
  return ((addr & 0x3ffff) >> 4) | (lead_bytes >> 4) << 16;
}
constexpr uint32_t kTcDescHigh = (1024u >> 4) | 1u << 14 | 2u << 29;
// fp32 accumulators, bf16 operands, M = 128; B read along the rows or, ACROSS, across them
template <bool ACROSS>
__device__ __forceinline__ uint32_t tc_idesc(int n) {
  return 1u << 4 | 1u << 7 | 1u << 10 | (ACROSS ? 1u << 16 : 0u) | (uint32_t)(n / 8) << 17 | (128u / 16) << 24;
}

// Columns of tensor memory.  Regions are used again within a chunk once what they held has been read.
enum : uint32_t {
  kTcS = 0,          // pieces of S (3 x DKP / 2)
  kTcU = 0,          //   then of U (PP x 32);  backward: of Y (3 x 32)
  kTcLU = 96,        //   and of what updates the state (3 x 32)
  kTcD = 192,        // K S (64), then T X (64), then the state's update (DKP)
  kTcD2 = 256,       //   backward: beside K dS' the product P^T dO (64)
  kTcO = 320,        // Q S (64);  backward: pieces of dO (NP x 32)
  kTcX = 384,        // pieces of X (3 x 32), then P U (64)
  kTcG = 416,        // backward: pieces of scale e^G dO (3 x 32)
  kTcCols = 512
};

template <int NP, int DKP, int PP>
struct alignas(1024) TcStage {
  __nv_bfloat16 k[NP][kC * DKP], q[NP][kC * DKP];
  __nv_bfloat16 t[3][kTri], pm[PP][kTri];
  float vec[kVec];
};
template <int NP, int DKP, int PP>
struct alignas(1024) TcSmem {
  static constexpr int kRowUnits = NP == 1 ? 4 : 2;      // 16-byte units of a row that pass at a time
  TcStage<NP, DKP, PP> stage[2];
  float4 rows[16][32 * kRowUnits];                       // per warp, see tc_store_rows
  int first[2][128];             // by chunk parity: a channel's first position that is not finite, or kC
  uint64_t full[2];              // a stage's tiles are there
  uint64_t ready[3], done[3];    // operands of a round are in tensor memory; its products are finished
  uint32_t tmem;
};

constexpr int kTcThreads = 512 + 32;

// ---- products, issued by one warp -------------------------------------------------------------
// Which products of pieces: LOW: index sums 1 .. MAXI; else the leading one.
// d (N columns) += A (NA pieces, K / 2 columns apart) x tile of NB pieces, over K / 16 steps.
//   FULL   B [n][k] of 64 rows, K = DKP: both halves of a (kC x DKP) tile
//   ACROSS B [k][n], K = 64, N = DKP
//   LOWER  B [n][k], K = 64, N = 64, zero above the diagonal;  UPPER  the same read across, [k][n]
enum TcForm { kFull, kAcross, kLower, kUpper };
template <TcForm FORM, int NA, int NB, int MAXI, int DKP>
__device__ __forceinline__ void tc_product(uint32_t d, uint32_t a, uint32_t tile, bool lead, bool& started,
                                           uint32_t issue) {
  constexpr int kSteps = (FORM == kFull ? DKP : kC) / 16, kTile = (FORM == kLower || FORM == kUpper ? kTri : kC * DKP) * 2;
  const uint32_t base = tc_desc(tile, FORM == kAcross ? kC * 64 * 2 : 16);
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      if (i + j > MAXI || (i + j == 0) != lead) continue;
#pragma unroll
      for (int s0 = 0; s0 < kSteps; ++s0) {
        const int s = FORM == kUpper ? kSteps - 1 - s0 : s0;       // the step that covers all columns comes first
        const uint32_t as = a + i * (kSteps * 8) + s * 8, bt = base + j * (kTile / 16);
        if (FORM == kFull)
          tc_mma(d, as, bt + ((s >> 2) * (kC * 64 * 2) + (s & 3) * 32) / 16, kTcDescHigh, tc_idesc<false>(64), started, issue);
        else if (FORM == kAcross)
          tc_mma(d, as, bt + s * (2048 / 16), kTcDescHigh, tc_idesc<true>(DKP), started, issue);
        else if (FORM == kLower)         // columns from 16 s
          tc_mma(d + 16 * s, as, bt + s * ((2048 + 32) / 16), kTcDescHigh, tc_idesc<false>(kC - 16 * s), started, issue);
        else                             // columns below 16 (s + 1)
          tc_mma(d, as, bt + s * (2048 / 16), kTcDescHigh, tc_idesc<true>(16 * (s + 1)), started, issue);
        started = true;
      }
    }
}
template <TcForm FORM, int NA, int NB, int MAXI, int DKP>
__device__ __forceinline__ void tc_full_product(uint32_t d, uint32_t a, uint32_t tile, uint32_t issue) {
  bool started = false;
  tc_product<FORM, NA, NB, MAXI, DKP>(d, a, tile, false, started, issue);
  tc_product<FORM, NA, NB, MAXI, DKP>(d, a, tile, true, started, issue);
}

template <int NP, int DKP, int PP>
__device__ __forceinline__ void tc_load_stage(TcSmem<NP, DKP, PP>& s, const DeltaParams& p, int b, int h, int ch, int st) {
  const size_t at = ((size_t)b * p.Hv + h) * p.n + ch, atk = ((size_t)b * p.Hk + h / p.group) * p.n + ch;
  auto& g = s.stage[st];
  uint64_t* bar = &s.full[st];
  mbar_arrive_expect_tx(bar, sizeof(g.k) + sizeof(g.q) + sizeof(g.t) + sizeof(g.pm) + sizeof(g.vec));
  bulk_load(g.k, p.kimg + atk * (NP * kC * DKP), sizeof(g.k), bar);
  bulk_load(g.q, p.qimg + atk * (NP * kC * DKP), sizeof(g.q), bar);
  bulk_load(g.t, p.timg + at * (3 * kTri), sizeof(g.t), bar);
  bulk_load(g.pm, p.pimg + at * (3 * kTri), sizeof(g.pm), bar);
  bulk_load(g.vec, p.vec + at * kVec, sizeof(g.vec), bar);
}
template <typename Smem>
__device__ __forceinline__ Smem& tc_smem() {
  extern __shared__ unsigned char tc_raw[];
  return *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(tc_raw) + 1023) & ~uintptr_t(1023));
}
template <typename Smem>
__device__ __forceinline__ void tc_init(Smem& s) {
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) mbar_init(&s.full[i], 1);
    for (int i = 0; i < 3; ++i) {
      mbar_init(&s.ready[i], 16);
      mbar_init(&s.done[i], 1);
    }
    fence_mbar_init();
  }
  if (threadIdx.x >= 512) tc_alloc(&s.tmem, kTcCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
}
__device__ __forceinline__ void tc_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// This thread's part of a round's operands is written (and what it read of the last round's results is read).
__device__ __forceinline__ void tc_ready(uint64_t* bar) {
  tc_wait_store();
  tc_fence_before();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) tc_arrive(bar);
}

// The warp's 32 rows of N floats to a dense [row][pitch] array.  A thread holds a row, and 32 rows at a time are 32
// lines of memory per store; through shared memory (units permuted by the row) a store covers U units of 32 / U rows.
template <int U, int N>
__device__ __forceinline__ void tc_store_rows(float4* buf, float* base, int pitch, int rows, const float (&v)[N], int lane) {
  auto at = [](int r, int u) { return r * U + (u ^ (U == 8 ? r & 7 : U == 4 ? (r >> 1) & 3 : (r >> 2) & 1)); };
#pragma unroll
  for (int p0 = 0; p0 < N; p0 += 4 * U) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      buf[at(lane, u)] = make_float4(v[p0 + 4 * u], v[p0 + 4 * u + 1], v[p0 + 4 * u + 2], v[p0 + 4 * u + 3]);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int r = lane / U + i * (32 / U), u = lane % U;
      if (r < rows) *reinterpret_cast<float4*>(base + (size_t)r * pitch + p0 + 4 * u) = buf[at(r, u)];
    }
    __syncwarp();
  }
}
// 16 positions of one channel from / to a (positions, channels) tensor; neighbouring lanes are neighbouring channels.
template <typename T>
__device__ __forceinline__ void tc_load_col(const T* src, long long sl, int rows, bool live, T (&v)[16]) {
  if (rows >= 16 && live) {
#pragma unroll
    for (int i = 0; i < 16; ++i, src += sl) v[i] = *src;
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = live && i < rows ? src[i * sl] : from_f32<T>(0.0f);
  }
}
template <typename T>
__device__ __forceinline__ void tc_store_col(T* dst, long long sl, int rows, bool live, const float (&v)[16]) {
  if (rows >= 16 && live) {
#pragma unroll
    for (int i = 0; i < 16; ++i, dst += sl) *dst = from_f32<T>(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (live && i < rows) dst[i * sl] = from_f32<T>(v[i]);
  }
}
// f(i, vec[i]) for 16 consecutive factors, read four at a time
template <typename F>
__device__ __forceinline__ void tc_each(const float* vec, F f) {
#pragma unroll
  for (int i = 0; i < 16; i += 4) {
    const float4 x = *reinterpret_cast<const float4*>(vec + i);
    f(i, x.x);
    f(i + 1, x.y);
    f(i + 2, x.z);
    f(i + 3, x.w);
  }
}

// See is_bad: 16 positions from c0 of a channel.  What is not finite becomes 0, the first one is noted.
__device__ __forceinline__ void tc_note_bad(float (&x)[16], int* first, int c0) {
  float big = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; i += 2) big = max3_abs(big, x[i], x[i + 1]);
  if (!is_bad(big)) return;
#pragma unroll
  for (int i = 15; i >= 0; --i)
    if (is_bad(x[i])) {
      atomicMin(first, c0 + i);
      x[i] = 0.0f;
    }
}
__device__ __forceinline__ void tc_set_from(float (&x)[16], int first, int c0) {
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (c0 + i >= first) x[i] = quiet_nan();
}

// ---- forward ------------------------------------------------------------------------------------
template <typename T, int NP, int DKP, bool SAVE>
__global__ void __launch_bounds__(kTcThreads, 1) delta_fwd_tc(const __grid_constant__ DeltaParams p) {
  constexpr int PP = NP == 1 ? 2 : 3, QK = DKP / 4;
  using Smem = TcSmem<NP, DKP, PP>;
  Smem& s = tc_smem<Smem>();
  const int h = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  tc_init(s);
  const uint32_t tm = __shfl_sync(0xffffffffu, s.tmem, 0);
  Wait wait{p.err};
  if (warp == 16) {
    const uint32_t issue = lane == 0;
    for (int i = 0; issue && i < 2 && i < p.n; ++i) tc_load_stage(s, p, b, h, i, i);
    for (int ch = 0; ch < p.n; ++ch) {
      const int st = ch & 1, par = ch & 1;
      auto& g = s.stage[st];
      const uint32_t sk = smem_u32(g.k), sq = smem_u32(g.q), stt = smem_u32(g.t), sp = smem_u32(g.pm);
      wait(&s.full[st], (ch >> 1) & 1);
      wait(&s.ready[0], par);
      tc_fence_after();
      tc_full_product<kFull, 3, NP, 2, DKP>(tm + kTcD, tm + kTcS, sk, issue);
      tc_full_product<kFull, 3, NP, PP - 1, DKP>(tm + kTcO, tm + kTcS, sq, issue);
      if (issue) tc_commit(&s.done[0]);
      // every thread is past the last chunk, whose stage is free
      if (issue && !wait.dead && ch >= 1 && ch + 1 < p.n) tc_load_stage(s, p, b, h, ch + 1, st ^ 1);
      wait(&s.ready[1], par);
      tc_fence_after();
      tc_full_product<kLower, 3, 3, 2, DKP>(tm + kTcD, tm + kTcX, stt, issue);
      if (issue) tc_commit(&s.done[1]);
      wait(&s.ready[2], par);
      tc_fence_after();
      tc_full_product<kAcross, 3, NP, 2, DKP>(tm + kTcD, tm + kTcLU, sk, issue);
      tc_full_product<kLower, PP, PP, PP - 1, DKP>(tm + kTcX, tm + kTcU, sp, issue);
      if (issue) tc_commit(&s.done[2]);
    }
    __syncwarp();
  } else {
    const int quarter = warp >> 2, row = 32 * (warp & 3) + lane, d = 128 * blockIdx.x + row;
    const bool live = d < p.dvw;
    const int kept = p.dvp - (d - lane);           // rows of this warp that the saved arrays have
    const uint32_t my = tm + ((uint32_t)(32 * (warp & 3)) << 16);
    const size_t head = (size_t)b * p.Hv + h;
    const T* vb = static_cast<const T*>(p.v.ptr) + b * p.v.sb + h * p.v.sh + d;
    T* ob = static_cast<T*>(const_cast<void*>(p.o.ptr)) + b * p.o.sb + h * p.o.sh + d;
    float S[QK / 16][16];
    const float* h0 = p.h0 != nullptr ? p.h0 + head * p.dkw * p.dvw + d : nullptr;
#pragma unroll
    for (int i = 0; i < QK; ++i) {
      const int k = quarter * QK + i;
      S[i / 16][i % 16] = h0 != nullptr && live && k < p.dkw ? h0[(size_t)k * p.dvw] : 0.0f;
    }
    const int c0 = 16 * quarter;
    if (quarter == 0) s.first[0][row] = kC;        // the others read and write it behind the first round of products
    for (int ch = 0; ch < p.n; ++ch) {
      int* first = &s.first[ch & 1][row];
      const int st = ch & 1, par = ch & 1, rows = min(kC, p.L - ch * kC);
      const float* vec = s.stage[st].vec;
      const long long t0 = (long long)ch * kC + c0;
#pragma unroll
      for (int i = 0; i < QK / 16; ++i) tc_put<3>(my + kTcS + quarter * (QK / 2) + 8 * i, DKP / 2, S[i]);
      tc_ready(&s.ready[0]);
      T vr[16];
      tc_load_col(vb + t0 * p.v.sl, p.v.sl, rows - c0, live, vr);
      auto save = [&](int i) {                   // 16 columns of S, behind a round of products each: 478 -> 452 us
        if (SAVE)
          tc_store_rows<Smem::kRowUnits>(
              s.rows[warp], p.states + ((head * p.n + ch) * p.dvp + d - lane) * DKP + quarter * QK + 16 * i, DKP, kept, S[i], lane);
      };
      if (QK == 32) save(0);
      wait(&s.full[st], (ch >> 1) & 1);
      wait(&s.done[0], par);
      tc_fence_after();
      float x[16];
      tc_load_f32(my + kTcD + c0, x);
      tc_each(vec + c0, [&](int i, float eg) { x[i] = fmaf(-eg, x[i], to_f32(vr[i])); });
      tc_each(vec + 2 * kC + c0, [&](int i, float be) { x[i] *= be; });
      if (quarter == 0) s.first[(ch + 1) & 1][row] = kC;       // whose readers of the chunk before are done
      tc_note_bad(x, first, c0);
      tc_put<3>(my + kTcX + c0 / 2, kC / 2, x);
      tc_ready(&s.ready[1]);
      save(QK / 16 - 1);
      wait(&s.done[1], par);
      tc_fence_after();
      tc_load_f32(my + kTcD + c0, x);
      const int bad = *first;
      tc_put<PP>(my + kTcU + c0 / 2, kC / 2, x);
      // Without the branch where dk is 128 and states are saved (wide training 455 -> 439 us), with it elsewhere (128 heads of
      // 64 x 128: 176 -> 170, inference of 128 x 128: 193 -> 185): the schedules differ.
      if ((SAVE && DKP == 128) || bad < kC) tc_set_from(x, bad, c0);
      float y[16];
      tc_each(vec + kC + c0, [&](int i, float la) { y[i] = x[i] * la; });
      tc_put<3>(my + kTcLU + c0 / 2, kC / 2, y);
      tc_ready(&s.ready[2]);
      if (SAVE)
        tc_store_rows<Smem::kRowUnits>(s.rows[warp], p.us + ((head * p.n + ch) * p.dvp + d - lane) * kC + c0, kC, kept, x, lane);
      wait(&s.done[2], par);
      tc_fence_after();
      const float keep = vec[kC - 1];
#pragma unroll
      for (int j = 0; j < QK / 16; ++j) {
        tc_load_f32(my + kTcD + quarter * QK + 16 * j, x);
#pragma unroll
        for (int i = 0; i < 16; ++i) S[j][i] = fmaf(keep, S[j][i], x[i]);
      }
      tc_load_f32(my + kTcO + c0, y);
      tc_load_f32(my + kTcX + c0, x);
      tc_each(vec + c0, [&](int i, float eg) { x[i] = fmaf(p.scale * eg, y[i], x[i]); });
      if (bad < kC) tc_set_from(x, bad, c0);
      tc_store_col(ob + t0 * p.o.sl, p.o.sl, rows - c0, live, x);
    }
    if (p.last != nullptr && live) {
      float* last = p.last + head * p.dkw * p.dvw + d;
#pragma unroll
      for (int i = 0; i < QK; ++i) {
        const int k = quarter * QK + i;
        if (k < p.dkw) last[(size_t)k * p.dvw] = S[i / 16][i % 16];
      }
    }
    tc_fence_before();
  }
  wait.drain();
  __syncthreads();
  if (warp == 16) tc_free(tm, kTcCols);
}

// ---- backward, chunks in reverse ------------------------------------------------------------------
template <typename T, int NP, int DKP>
__global__ void __launch_bounds__(kTcThreads, 1) delta_bwd_tc(const __grid_constant__ DeltaParams p) {
  constexpr int QK = DKP / 4;
  using Smem = TcSmem<NP, DKP, 3>;
  Smem& s = tc_smem<Smem>();
  const int h = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  tc_init(s);
  const uint32_t tm = __shfl_sync(0xffffffffu, s.tmem, 0);
  Wait wait{p.err};
  if (warp == 16) {
    const uint32_t issue = lane == 0;
    for (int i = 0; issue && i < 2 && i < p.n; ++i) tc_load_stage(s, p, b, h, p.n - 1 - i, i);
    for (int it = 0; it < p.n; ++it) {
      const int st = it & 1, par = it & 1;
      auto& g = s.stage[st];
      const uint32_t sk = smem_u32(g.k), sq = smem_u32(g.q), stt = smem_u32(g.t), sp = smem_u32(g.pm);
      wait(&s.full[st], (it >> 1) & 1);
      wait(&s.ready[0], par);
      tc_fence_after();
      tc_full_product<kFull, 3, NP, 2, DKP>(tm + kTcD, tm + kTcS, sk, issue);
      tc_full_product<kUpper, NP, 3, 2, DKP>(tm + kTcD2, tm + kTcO, sp, issue);
      if (issue) tc_commit(&s.done[0]);
      if (issue && !wait.dead && it >= 1 && it + 1 < p.n) tc_load_stage(s, p, b, h, p.n - 2 - it, st ^ 1);
      wait(&s.ready[1], par);
      tc_fence_after();
      tc_full_product<kUpper, 3, 3, 2, DKP>(tm + kTcD, tm + kTcU, stt, issue);
      if (issue) tc_commit(&s.done[1]);
      wait(&s.ready[2], par);
      tc_fence_after();
      bool started = false;
      tc_product<kAcross, 3, NP, 2, DKP>(tm + kTcD, tm + kTcG, sq, false, started, issue);
      tc_product<kAcross, 3, NP, 2, DKP>(tm + kTcD, tm + kTcLU, sk, false, started, issue);
      tc_product<kAcross, 3, NP, 2, DKP>(tm + kTcD, tm + kTcG, sq, true, started, issue);
      tc_product<kAcross, 3, NP, 2, DKP>(tm + kTcD, tm + kTcLU, sk, true, started, issue);
      if (issue) tc_commit(&s.done[2]);
    }
    __syncwarp();
  } else {
    const int quarter = warp >> 2, row = 32 * (warp & 3) + lane, d = 128 * blockIdx.x + row;
    const bool live = d < p.dvw;
    const int kept = p.dvp - (d - lane);           // rows of this warp that the saved arrays have
    const uint32_t my = tm + ((uint32_t)(32 * (warp & 3)) << 16);
    const size_t head = (size_t)b * p.Hv + h;
    const T* gb = static_cast<const T*>(p.o.ptr) + b * p.o.sb + h * p.o.sh + d;
    T* ob = static_cast<T*>(const_cast<void*>(p.dv.ptr)) + b * p.dv.sb + h * p.dv.sh + d;
    const int c0 = 16 * quarter;
    float S[QK / 16][16];
    const float* h0 = p.h0 != nullptr ? p.h0 + head * p.dkw * p.dvw + d : nullptr;
#pragma unroll
    for (int i = 0; i < QK; ++i) {
      const int k = quarter * QK + i;
      S[i / 16][i % 16] = h0 != nullptr && live && k < p.dkw ? h0[(size_t)k * p.dvw] : 0.0f;
    }
    T gr[16];
    auto fetch = [&](int ch) {
      tc_load_col(gb + ((long long)ch * kC + c0) * p.o.sl, p.o.sl, p.L - ch * kC - c0, live, gr);
    };
    auto put_grad = [&] {
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = to_f32(gr[i]);
      tc_put<NP>(my + kTcO + c0 / 2, kC / 2, x);
    };
    fetch(p.n - 1);
    put_grad();
    for (int it = 0; it < p.n; ++it) {
      const int ch = p.n - 1 - it, st = it & 1, par = it & 1, rows = min(kC, p.L - ch * kC);
      const float* vec = s.stage[st].vec;
      const long long t0 = (long long)ch * kC + c0;
      float x[16];
#pragma unroll
      for (int i = 0; i < QK / 16; ++i) tc_put<3>(my + kTcS + quarter * (QK / 2) + 8 * i, DKP / 2, S[i]);
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = to_f32(gr[i]);
      wait(&s.full[st], (it >> 1) & 1);
      tc_each(vec + c0, [&](int i, float eg) { x[i] *= p.scale * eg; });
      tc_put<3>(my + kTcG + c0 / 2, kC / 2, x);
      tc_ready(&s.ready[0]);
      if (NP == 3 && ch > 0) fetch(ch - 1);
      float* dst = p.dstates + ((head * p.n + ch) * p.dvp + d - lane) * DKP + quarter * QK;
#pragma unroll
      for (int i = 0; i < QK / 16; ++i) tc_store_rows<Smem::kRowUnits>(s.rows[warp], dst + 16 * i, DKP, kept, S[i], lane);
      wait(&s.done[0], par);
      tc_fence_after();
      float y[16];
      tc_load_f32(my + kTcD + c0, x);
      tc_load_f32(my + kTcD2 + c0, y);
      tc_each(vec + kC + c0, [&](int i, float la) { x[i] = fmaf(la, x[i], y[i]); });
      tc_put<3>(my + kTcU + c0 / 2, kC / 2, x);
      tc_ready(&s.ready[1]);
      if (NP == 1 && ch > 0) fetch(ch - 1);      // behind the shorter wait; 32-bit values would spill (67 -> 72 us)
      wait(&s.done[1], par);
      tc_fence_after();
      tc_load_f32(my + kTcD + c0, x);
      float z[16];
      tc_each(vec + 2 * kC + c0, [&](int i, float be) { z[i] = x[i] * be; });
      tc_each(vec + c0, [&](int i, float eg) { y[i] = -eg * z[i]; });
      tc_put<3>(my + kTcLU + c0 / 2, kC / 2, y);
      tc_ready(&s.ready[2]);
      tc_store_rows<Smem::kRowUnits>(s.rows[warp], p.dxs + ((head * p.n + ch) * p.dvp + d - lane) * kC + c0, kC, kept, x, lane);
      tc_store_col(ob + t0 * p.dv.sl, p.dv.sl, rows - c0, live, z);
      const float keep = vec[kC - 1];
      if (ch > 0) put_grad();
      wait(&s.done[2], par);
      tc_fence_after();
#pragma unroll
      for (int j = 0; j < QK / 16; ++j) {
        tc_load_f32(my + kTcD + quarter * QK + 16 * j, x);
#pragma unroll
        for (int i = 0; i < 16; ++i) S[j][i] = fmaf(keep, S[j][i], x[i]);
      }
    }
    if (p.last != nullptr && live) {
      float* last = p.last + head * p.dkw * p.dvw + d;
#pragma unroll
      for (int i = 0; i < QK; ++i) {
        const int k = quarter * QK + i;
        if (k < p.dkw) last[(size_t)k * p.dvw] = S[i / 16][i % 16];
      }
    }
    tc_fence_before();
  }
  wait.drain();
  __syncthreads();
  if (warp == 16) tc_free(tm, kTcCols);
}

}  // namespace ssm
