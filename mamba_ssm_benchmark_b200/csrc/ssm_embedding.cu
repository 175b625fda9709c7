// ssm_embedding.cu — rows of a table by token, scaled, and the table's gradient.
//
//   y[t] = scale W[idx[t]],   dW[v] = scale sum over t with idx[t] = v of dy[t]
// Both directions are bound by memory: the rows that are read and written.  The gradient's places are sorted by token
// (stable, so that a token's places stay in order), cut into chunks of nearly equal length whatever the tokens'
// frequencies, and summed chunk by chunk: fp32 within a chunk (up to 127 places, below), fp64 over the chunks that a frequent
// token spans.  No atomics on floats, a fixed order: results are reproducible.  Rows that no token names are zeroed by CTAs of
// the same launch.
//
// 65536 x 2560 bf16 of 50257 words: forward 68 us (5.7 TB/s of what is read from memory and written), sort 21, sums 103 (DRAM
// at 67 % of its rate, 5.5 TB/s), long runs 12.  One CTA to a token instead of chunks would have the most frequent one, a
// tenth of all places, decide; chunks that cut short runs cost 25 us more for their partial rows.
//
// A token outside 0 .. V-1 gives a row of NaN and no gradient, and sets bit 1 of the device error word.
#include <cooperative_groups.h>

#include <algorithm>
#include <cstdio>

#include "ssm_b200.h"
#include "ssm_launch.cuh"
#include "ssm_rows.cuh"

namespace cg = cooperative_groups;

namespace ssm {
int report_error(int code, const char* msg);
int* device_error_word();
}  // namespace ssm

namespace {

using ssm::Slot;
using ssm::add2;
using ssm::bc2;
using ssm::mul2;
using ssm::from_f32;
using ssm::to_f32;

constexpr int kBadToken = 2;        // bit of the device error word

struct EmbedParams {
  const void* idx;
  int idx8;                         // 64-bit ids
  const void* w;                    // table, or the gradient of the rows
  void* y;                          // rows, or the gradient of the table
  long long ws, ys;                 // row strides
  long long T, V;
  int C;
  float scale;
  int* err;
  // backward
  const uint2* sorted;              // (token, place) by token
  float* part;                      // (chunks, 2, C)
  long long chunks;
  int len;                          // places to a chunk
  int slabs;                        // CTAs over the channels
  int* joins;                       // how many chunks a run goes on from, then which
  uint32_t* named;                  // a bit for every token: it occurs
};

__device__ __forceinline__ long long token_at(const EmbedParams& p, long long t) {
  return p.idx8 ? static_cast<const long long*>(p.idx)[t] : (long long)static_cast<const int*>(p.idx)[t];
}

// ---- forward ----------------------------------------------------------------------------------
// A warp takes kAhead units a lane of one row, so that as many loads are on their way; a row has `pieces` warps.
constexpr int kAhead = 4;
template <typename T, bool RAGGED, bool SCALE>
__global__ void __launch_bounds__(256) embed_fwd(const __grid_constant__ EmbedParams p, int pieces) {
  constexpr int VEC = 16 / sizeof(T);
  using Part = Slot<T, VEC, RAGGED>;
  ssm::pdl_launch_dependents();
  ssm::pdl_wait();
  const long long item = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const long long t = item / pieces;
  if (t >= p.T) return;
  const int lane = threadIdx.x & 31, c0 = (int)(item - t * pieces) * kAhead * Part::kTaken;
  const long long v = token_at(p, t);
  const bool bad = v < 0 || v >= p.V;
  if (bad && lane == 0 && p.err != nullptr) atomicOr(p.err, kBadToken);
  const T* row = static_cast<const T*>(p.w) + (bad ? 0 : v) * p.ws;
  T* out = static_cast<T*>(p.y) + t * p.ys;
  uint4 raw[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; ++k) raw[k] = Part::take(row, c0 + k * Part::kTaken, p.C, lane);
#pragma unroll
  for (int k = 0; k < kAhead; ++k) {
    const int c = c0 + k * Part::kTaken;
    if (c >= p.C) continue;                            // the same for the warp
    uint32_t w[4];
    Part::taken(raw[k], row, c, w);
    if (SCALE || bad) {
      float2 x[VEC / 2];
      Part::unpack(w, x);
      const float2 scale = bc2(bad ? __int_as_float(0x7fc00000) : p.scale);
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) x[i] = bad ? scale : mul2(x[i], scale);
      Part::pack(x, w);
    }
    Part::write(out, c, min(p.C, c + Part::kTaken), lane, w);
  }
}

// ---- places by token ----------------------------------------------------------------------------
// A stable radix sort, kDigit bits a pass, by one cluster: with a launch a step it would be six launches.  A warp
// owns consecutive places; counts are kept by warp, so that its places land in order behind those of the warps before it.
constexpr int kDigit = 9, kBins = 1 << kDigit, kSortWarps = 32, kHeld = 8;
struct SortSmem {
  uint32_t count[kSortWarps][kBins];   // by warp: counts, then where its next place of a bin goes
  uint32_t total[kBins];               // of this CTA
  uint32_t base[kBins];
  uint32_t warp_sum[kSortWarps];
};

__global__ void __launch_bounds__(1024) embed_sort(const __grid_constant__ EmbedParams p, uint2* a, uint2* b, int passes) {
  extern __shared__ __align__(16) unsigned char raw[];
  SortSmem& s = *reinterpret_cast<SortSmem*>(raw);
  ssm::pdl_launch_dependents();
  ssm::pdl_wait();
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (rank == 0 && threadIdx.x == 0) p.joins[0] = 0;
  for (long long w = rank * 1024 + threadIdx.x; w < (p.V + 31) / 32; w += ctas * 1024) p.named[w] = 0;
  cluster.sync();
  // places of this warp: a multiple of 32 to each
  const long long per = ((p.T + ctas * kSortWarps - 1) / (ctas * kSortWarps) + 31) / 32 * 32;
  const long long first = min(p.T, (long long)(rank * kSortWarps + warp) * per), last = min(p.T, first + per);
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * kDigit;
    const uint2* src = pass & 1 ? a : b;               // from the second pass on
    uint2* dst = pass & 1 ? b : a;
    auto item = [&](long long t) {
      if (pass > 0) return src[t];
      const long long v = token_at(p, t);
      return make_uint2((uint32_t)(v < 0 || v >= p.V ? p.V : v), (uint32_t)t);
    };
    // up to kHeld places a lane stay in registers, loaded at once
    const bool held = per <= 32 * kHeld;
    uint2 x[kHeld];
    if (held) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i) x[i] = item(min(first + 32 * i + lane, p.T - 1));      // no branch between the loads
    }
    for (int i = threadIdx.x; i < kSortWarps * kBins / 4; i += 1024) reinterpret_cast<uint4*>(s.count)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    auto count = [&](uint32_t token) { atomicAdd(&s.count[warp][token >> shift & (kBins - 1)], 1u); };
    if (held) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i)
        if (first + 32 * i + lane < last) count(x[i].x);
    } else {
#pragma unroll 4
      for (long long t = first + lane; t < last; t += 32) count(item(t).x);
    }
    __syncthreads();
    // by bin: this CTA's total
    uint32_t mine = 0;
    if (threadIdx.x < kBins) {
      for (int w = 0; w < kSortWarps; ++w) mine += s.count[w][threadIdx.x];
      s.total[threadIdx.x] = mine;
    }
    cluster.sync();
    // by bin: what the CTAs before have of it, and all CTAs have
    uint32_t before = 0, all = 0;
    if (threadIdx.x < kBins)
      for (int r = 0; r < ctas; ++r) {
        const uint32_t n = cluster.map_shared_rank(s.total, r)[threadIdx.x];
        if (r < rank) before += n;
        all += n;
      }
    uint32_t run = all;                                // inclusive sum over the bins
#pragma unroll
    for (int m = 1; m < 32; m *= 2) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, run, m);
      if (lane >= m) run += up;
    }
    if (lane == 31) s.warp_sum[warp] = run;
    __syncthreads();
    if (threadIdx.x < kBins) {
      uint32_t at = run - all + before;
      for (int w = 0; w < warp; ++w) at += s.warp_sum[w];
      for (int w = 0; w < kSortWarps; ++w) {
        const uint32_t n = s.count[w][threadIdx.x];
        s.count[w][threadIdx.x] = at;
        at += n;
      }
    }
    __syncthreads();
    auto place = [&](bool live, uint2 v) {
      const uint32_t bin = live ? v.x >> shift & (kBins - 1) : kBins;      // lanes past the end share a bin of their own
      // the lanes of the same bin, bit by bit (__match_any_sync takes its time by the number of values: 65536 places of
      // mostly different bins 8.2 us, this way 6.3)
      uint32_t same = 0xffffffffu;
#pragma unroll
      for (int i = 0; i <= kDigit; ++i) {
        const uint32_t set = __ballot_sync(0xffffffffu, bin >> i & 1);
        same &= bin >> i & 1 ? set : ~set;
      }
      const uint32_t to = live ? s.count[warp][bin] + __popc(same & ((1u << lane) - 1)) : 0;
      __syncwarp();
      if (live && lane == __ffs(same) - 1) s.count[warp][bin] += __popc(same);
      __syncwarp();
      if (live) dst[to] = v;
    };
    if (held) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i)
        if (first + 32 * i < last) place(first + 32 * i + lane < last, x[i]);
    } else {
#pragma unroll 2
      for (long long t0 = first; t0 < last; t0 += 32) {
        const bool live = t0 + lane < last;
        place(live, live ? item(t0 + lane) : make_uint2(0, 0));
      }
    }
    __threadfence();
    cluster.sync();                                    // the next pass reads what every CTA wrote, and counts anew
  }
  // a bit for every token that occurs, where its places start
  const uint2* out = passes & 1 ? a : b;
  const uint32_t none = 0xffffffffu;
  for (long long t = rank * 1024 + threadIdx.x; t < p.T; t += ctas * 1024) {
    const uint32_t v = out[t].x, before = t > 0 ? out[t - 1].x : none;
    if (v != before && v < p.V) atomicOr(p.named + (v >> 5), 1u << (v & 31));
  }
}

// ---- sums of the sorted places ---------------------------------------------------------------------
constexpr int kSumThreads = 256, kLongest = 64, kRows = 8, kFill = 32;      // kFill: a word of `named`

// Chunk q starts at the first place from q len on where another token begins, or at q len inside a run of more than len: it has
// up to 2 len - 1 places, all of which may be one token's, 126 additions of a fp32 sum.
// The sum of a run of equal tokens goes to the table where the chunk holds all of it, else to the chunk's partial
// rows: 0 where the run comes from the chunk before, 1 where it starts here and goes on.
template <typename T, bool RAGGED>
__global__ void __launch_bounds__(kSumThreads) embed_sum(const __grid_constant__ EmbedParams p) {
  __shared__ uint2 near[2 * kLongest + 1];             // from the place before the chunk's first possible one
  __shared__ int bound[2];
  ssm::pdl_launch_dependents();
  ssm::pdl_wait();
  constexpr int VEC = 16 / sizeof(T);
  using Part = Slot<T, VEC, RAGGED>;
  const int lane = threadIdx.x & 31;
  const int c0 = ((int)(blockIdx.x % p.slabs) * (blockDim.x >> 5) + (threadIdx.x >> 5)) * Part::kTaken;      // the warp's channels
  const int c1 = min(p.C, c0 + Part::kTaken);
  const long long item = blockIdx.x / p.slabs;
  constexpr uint32_t kNone = 0xffffffffu;
  // Chunks to sum and rows to zero take turns, so that reads and writes mix.
  const long long fills = (p.V + kFill - 1) / kFill, items = p.chunks + fills;
  const long long fill = item * fills / items, chunk = item - fill;
  if ((item + 1) * fills / items > fill) {             // rows without a token
    const uint32_t named = p.named[fill];
    const int rows = (int)min((long long)kFill, p.V - fill * kFill);
    const uint32_t zero[4] = {0, 0, 0, 0};
    if (c0 < p.C)
      for (int i = 0; i < rows; ++i)
        if (!(named >> i & 1)) Part::write(static_cast<T*>(p.y) + (fill * kFill + i) * p.ys, c0, c1, lane, zero);
    return;
  }
  const long long t0 = chunk * p.len;
  for (int i = threadIdx.x; i < 2 * p.len + 1; i += blockDim.x)
    near[i] = t0 - 1 + i >= 0 && t0 - 1 + i < p.T ? p.sorted[t0 - 1 + i] : make_uint2(kNone, 0);
  __syncthreads();
  // where this chunk and the next one start, from t0 on
  for (int side = 0; side < 2; ++side) {
    const int from = side * p.len, left = (int)min((long long)p.len, p.T - t0 - from);     // places that may start it
    if ((int)threadIdx.x < 32) {
      int at = kLongest;
      for (int i = threadIdx.x; i < left; i += 32)
        if (near[from + i].x != near[from + i + 1].x) at = min(at, i);
      at = __reduce_min_sync(0xffffffffu, at);
      if (threadIdx.x == 0) bound[side] = from + (t0 + from == 0 || at == kLongest ? 0 : at);
    }
  }
  __syncthreads();
  const int first = bound[0], n = (int)min((long long)bound[1], p.T - t0) - first;
  const uint2* at = near + 1 + first;                  // the chunk's places
  const uint32_t outer[2] = {at[-1].x, first + n < 2 * p.len && t0 + first + n < p.T ? at[n].x : kNone};
  if (threadIdx.x == 0 && blockIdx.x % p.slabs == 0) {
    const uint32_t v = at[n - 1].x;
    if (v < p.V && outer[1] == v && !(at[0].x == v && outer[0] == v)) p.joins[1 + atomicAdd(p.joins, 1)] = (int)chunk;
  }
  if (c0 >= p.C) return;
  float2 acc[VEC / 2] = {};
  int start = 0;                                       // of the run
  auto flush = [&](int end) {
    const uint32_t v = at[start].x;
    if (v < p.V) {
      const bool from = start == 0 && outer[0] == v, to = end == n && outer[1] == v;
      if (!from && !to) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) acc[i] = mul2(acc[i], bc2(p.scale));
        Part::pack(acc, w);
        Part::write(static_cast<T*>(p.y) + (long long)v * p.ys, c0, c1, lane, w);
      } else {
        float* out = p.part + ((size_t)chunk * 2 + (from ? 0 : 1)) * p.C;
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
          const int c = c0 + lane * VEC + 2 * i;
          if (c < c1) out[c] = acc[i].x;
          if (c + 1 < c1) out[c + 1] = acc[i].y;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) acc[i] = make_float2(0.0f, 0.0f);
    start = end;
  };
  auto row = [&](int i) { return static_cast<const T*>(p.w) + (long long)at[i].y * p.ws; };
  for (int i0 = 0; i0 < n; i0 += kRows) {
    uint4 raw[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      if (i0 + i < n) raw[i] = Part::take(row(i0 + i), c0, p.C, lane);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      if (i0 + i >= n) break;
      if (at[i0 + i].x != at[start].x) flush(i0 + i);
      uint32_t w[4];
      float2 x[VEC / 2];
      Part::taken(raw[i], row(i0 + i), c0, w);
      Part::unpack(w, x);
#pragma unroll
      for (int j = 0; j < VEC / 2; ++j) acc[j] = add2(acc[j], x[j]);
    }
  }
  flush(n);
}

// Runs that span chunks: the chunk where one starts is in the list (in any order), and adds what the next ones have of it.
// A warp has a partial row's 128 channels, the CTA's warps every eighth of the chunks, whose sums are added in order.
constexpr int kJoinWarps = 8;
template <typename T>
__global__ void __launch_bounds__(32 * kJoinWarps) embed_join(const __grid_constant__ EmbedParams p) {
  __shared__ double red[kJoinWarps][128];
  ssm::pdl_launch_dependents();
  ssm::pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, pieces = (p.C + 127) / 128;
  const long long items = (long long)p.joins[0] * pieces;
  for (long long item = blockIdx.x; item < items; item += gridDim.x) {
    const long long chunk = p.joins[1 + item / pieces];
    const int c0 = (int)(item % pieces) * 128;
    const uint32_t v = p.sorted[(chunk + 1) * p.len].x;
    long long end = chunk + 1;                         // the first chunk that does not start inside the run
    for (bool all = true; all;) {
      const long long q = end + threadIdx.x;
      const int n = __syncthreads_count(q < p.chunks && p.sorted[min((q + 1) * p.len, p.T) - 1].x == v);
      end += n;
      all = n == 32 * kJoinWarps;
    }
    double sum[4] = {};
    auto add = [&](const float* row) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c0 + lane + 32 * i < p.C) sum[i] += (double)row[c0 + lane + 32 * i];
    };
    if (warp == 0) add(p.part + ((size_t)chunk * 2 + 1) * p.C);
#pragma unroll 4
    for (long long q = chunk + 1 + warp; q < end; q += kJoinWarps) add(p.part + (size_t)q * 2 * p.C);
#pragma unroll
    for (int i = 0; i < 4; ++i) red[warp][lane + 32 * i] = sum[i];
    __syncthreads();
    if (threadIdx.x < 128 && c0 + threadIdx.x < p.C) {
      double s = 0.0;
      for (int w = 0; w < kJoinWarps; ++w) s += red[w][threadIdx.x];
      static_cast<T*>(p.y)[(long long)v * p.ys + c0 + threadIdx.x] = from_f32<T>((float)(s * (double)p.scale));
    }
    __syncthreads();
  }
}

// ---- host -----------------------------------------------------------------------------------
int fail(int code, const char* fmt, long long a = 0, long long b = 0) {
  char msg[256];
  snprintf(msg, sizeof(msg), fmt, a, b);
  return ssm::report_error(code, msg);
}
long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }
size_t round256(size_t x) { return (x + 255) & ~size_t(255); }

int check_shape(int64_t T, int64_t V, int64_t C) {
  if (T < 1 || V < 1 || C < 1) return fail(SSM_ERR_INVALID, "embedding: tokens, vocabulary and channels must be positive");
  if (T > (1LL << 30) || V > (1LL << 30) || C > (1LL << 20))
    return fail(SSM_ERR_INVALID, "embedding: shape out of range (tokens %lld, vocabulary %lld)", T, V);
  return SSM_OK;
}
int check_side(const char* what, const ssm_view& v) {
  char msg[128];
  if (v.ptr == nullptr) {
    snprintf(msg, sizeof(msg), "embedding: %s is required", what);
    return ssm::report_error(SSM_ERR_INVALID, msg);
  }
  if (v.dtype != SSM_F32 && v.dtype != SSM_BF16) {
    snprintf(msg, sizeof(msg), "embedding: %s must be float32 or bfloat16", what);
    return ssm::report_error(SSM_ERR_DTYPE, msg);
  }
  return SSM_OK;
}
// Whether the rows of both tensors are whole 16 bytes that start at multiples of 16.
bool aligned(int64_t C, int es, const ssm_view& a, const ssm_view& b) {
  auto fits = [&](const ssm_view& v) { return reinterpret_cast<uintptr_t>(v.ptr) % 16 == 0 && v.batch_stride * es % 16 == 0; };
  return C * es % 16 == 0 && fits(a) && fits(b);
}
// Channels of a warp, by a unit of 16 bytes to a lane.
int warp_channels(int es, bool ragged) { return (ragged ? 31 : 32) * 16 / es; }

template <typename T, bool RAGGED>
cudaError_t run_fwd(const EmbedParams& p, cudaStream_t st) {
  const int pieces = (int)ceil_div(p.C, warp_channels(sizeof(T), RAGGED) * kAhead);
  const unsigned grid = (unsigned)ceil_div(p.T * pieces, 8);
  return ssm::launch_pdl(p.scale == 1.0f ? embed_fwd<T, RAGGED, false> : embed_fwd<T, RAGGED, true>, grid, 256, 0, st, p, pieces);
}
template <typename T, bool RAGGED>
cudaError_t run_bwd(EmbedParams p, cudaStream_t st) {
  // as few CTAs over the channels as there can be, with warps in equal parts
  const long long warps = ceil_div(p.C, warp_channels(sizeof(T), RAGGED));
  p.slabs = (int)ceil_div(warps, kSumThreads / 32);
  const int threads = (int)ceil_div(warps, p.slabs) * 32;
  const unsigned grid = (unsigned)((p.chunks + ceil_div(p.V, kFill)) * p.slabs);
  cudaError_t e = ssm::launch_pdl(embed_sum<T, RAGGED>, grid, threads, 0, st, p);
  if (e == cudaSuccess && p.chunks > 1) {
    const long long most = (p.chunks - 1) * ceil_div(p.C, 128);
    e = ssm::launch_pdl(embed_join<T>, (unsigned)std::min<long long>(most, 148 * 4), 32 * kJoinWarps, 0, st, p);
  }
  return e;
}
template <typename T>
cudaError_t run(const EmbedParams& p, bool bwd, bool ragged, cudaStream_t st) {
  if (ragged) return bwd ? run_bwd<T, true>(p, st) : run_fwd<T, true>(p, st);
  return bwd ? run_bwd<T, false>(p, st) : run_fwd<T, false>(p, st);
}

// Places to a chunk: as many as leave every SM a dozen CTAs, 8 to kLongest.
int chunk_len(int64_t T, int64_t C) {
  const long long slabs = ceil_div(C, kSumThreads * 4);
  return (int)std::max<long long>(8, std::min<long long>(kLongest, T * slabs / (148 * 12)));
}

int run_sort(const EmbedParams& p, uint2* a, uint2* b, int passes, cudaStream_t st) {
  // With few places the barriers of a cluster cost as much as its CTAs save; with many their scattered stores, one a clock and SM,
  // take most of the time.  Forward and gradient of 50257 words of 16 channels in a graph, us with one, eight and sixteen CTAs:
  // 512 places 20.5, 21.9, 23.6; 1024: 22.6, 22.7, 24.6; 4096: 28.7, 24.6, 26.7; 16384: 68.9, 29.6, 29.9; 32768: 122, 39.1, 37.3;
  // 65536: 225, 57, 51.
  const int ctas = p.T <= 1024 ? 1 : p.T <= 16384 ? 8 : 16;
  ssm::ctas_per_sm<embed_sort>(1024, sizeof(SortSmem));
  if (ctas > 8) {
    const cudaError_t e = cudaFuncSetAttribute(embed_sort, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return fail(SSM_ERR_CUDA, "embedding: the sort's cluster is refused (error %lld)", (long long)e);
  }
  const cudaError_t e = ssm::launch_pdl_cluster(embed_sort, ctas, 1024, ctas, sizeof(SortSmem), st, p, a, b, passes);
  return e == cudaSuccess ? SSM_OK : fail(SSM_ERR_CUDA, "embedding: the sort's launch failed (error %lld)", (long long)e);
}

}  // namespace

extern "C" {

int ssm_embedding_fwd(int64_t T, int64_t V, int64_t C, const void* idx, int32_t idx_bytes, ssm_view weight, float scale,
                      ssm_view y, void* stream) {
  if (int rc = check_shape(T, V, C)) return rc;
  if (idx == nullptr || (idx_bytes != 4 && idx_bytes != 8))
    return fail(idx == nullptr ? SSM_ERR_INVALID : SSM_ERR_DTYPE, "embedding: the ids are required, in 32 or 64 bits");
  if (int rc = check_side("weight", weight)) return rc;
  if (int rc = check_side("y", y)) return rc;
  if (weight.dtype != y.dtype) return fail(SSM_ERR_DTYPE, "embedding: y must have the weight's dtype");
  EmbedParams p = {};
  p.idx = idx;
  p.idx8 = idx_bytes == 8;
  p.w = weight.ptr;
  p.ws = weight.batch_stride;
  p.y = const_cast<void*>(y.ptr);
  p.ys = y.batch_stride;
  p.T = T;
  p.V = V;
  p.C = (int)C;
  p.scale = scale;
  p.err = ssm::device_error_word();
  const int es = weight.dtype == SSM_BF16 ? 2 : 4;
  const bool ragged = !aligned(C, es, weight, y);
  if (ceil_div(T * ceil_div(C, warp_channels(es, ragged) * kAhead), 8) > 0x7fffffffLL)
    return fail(SSM_ERR_INVALID, "embedding: shape out of range (tokens %lld, channels %lld)", T, C);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = es == 2 ? run<__nv_bfloat16>(p, false, ragged, st) : run<float>(p, false, ragged, st);
  return e == cudaSuccess ? SSM_OK : fail(SSM_ERR_CUDA, "embedding forward launch failed (error %lld)", (long long)e);
}

int ssm_embedding_bwd_workspace_size(int64_t T, int64_t V, int64_t C, size_t* bytes) {
  if (bytes == nullptr) return fail(SSM_ERR_INVALID, "embedding: bytes is NULL");
  if (int rc = check_shape(T, V, C)) return rc;
  const size_t chunks = (size_t)ceil_div(T, chunk_len(T, C));
  *bytes = 2 * round256((size_t)T * sizeof(uint2)) + round256((chunks + 1) * sizeof(int)) +
           round256((size_t)ceil_div(V, 32) * sizeof(int)) + chunks * 2 * C * sizeof(float) + 256;
  return SSM_OK;
}

int ssm_embedding_bwd(int64_t T, int64_t V, int64_t C, const void* idx, int32_t idx_bytes, float scale, ssm_view dy,
                      ssm_view dweight, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_shape(T, V, C)) return rc;
  if (idx == nullptr || (idx_bytes != 4 && idx_bytes != 8))
    return fail(idx == nullptr ? SSM_ERR_INVALID : SSM_ERR_DTYPE, "embedding: the ids are required, in 32 or 64 bits");
  if (int rc = check_side("dy", dy)) return rc;
  if (int rc = check_side("dweight", dweight)) return rc;
  if (dy.dtype != dweight.dtype) return fail(SSM_ERR_DTYPE, "embedding: dweight must have dy's dtype");
  size_t need = 0;
  ssm_embedding_bwd_workspace_size(T, V, C, &need);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(SSM_ERR_WORKSPACE, "embedding: workspace of %lld bytes required, %lld given", (long long)need,
                (long long)workspace_bytes);
  EmbedParams p = {};
  p.idx = idx;
  p.idx8 = idx_bytes == 8;
  p.w = dy.ptr;
  p.ws = dy.batch_stride;
  p.y = const_cast<void*>(dweight.ptr);
  p.ys = dweight.batch_stride;
  p.T = T;
  p.V = V;
  p.C = (int)C;
  p.scale = scale;
  p.len = chunk_len(T, C);
  p.chunks = ceil_div(T, p.len);
  const int es = dy.dtype == SSM_BF16 ? 2 : 4;
  const bool ragged = !aligned(C, es, dy, dweight);
  if ((p.chunks + ceil_div(V, kFill)) * ceil_div(C, warp_channels(es, ragged)) > 0x7fffffffLL)
    return fail(SSM_ERR_INVALID, "embedding: shape out of range (tokens %lld, channels %lld)", T, C);
  unsigned char* at = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~uintptr_t(255));
  uint2* a = reinterpret_cast<uint2*>(at);
  uint2* b = reinterpret_cast<uint2*>(at + round256((size_t)T * sizeof(uint2)));
  at += 2 * round256((size_t)T * sizeof(uint2));
  p.joins = reinterpret_cast<int*>(at);
  at += round256((size_t)(p.chunks + 1) * sizeof(int));
  p.named = reinterpret_cast<uint32_t*>(at);
  p.part = reinterpret_cast<float*>(at + round256((size_t)ceil_div(V, 32) * sizeof(int)));
  int passes = 1;                                      // of kDigit bits, for the ids 0 .. V (V: outside)
  while (passes * kDigit < 32 && (V >> (passes * kDigit)) > 0) ++passes;
  p.sorted = passes & 1 ? a : b;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (int rc = run_sort(p, a, b, passes, st)) return rc;
  const cudaError_t e = es == 2 ? run<__nv_bfloat16>(p, true, ragged, st) : run<float>(p, true, ragged, st);
  return e == cudaSuccess ? SSM_OK : fail(SSM_ERR_CUDA, "embedding backward launch failed (error %lld)", (long long)e);
}

}  // extern "C"
