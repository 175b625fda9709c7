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
// Up to kList tokens: a thread each, sorted by rank in registers.  More: a cluster of up to eight CTAs shares a row, a slice
// of tokens each, kept in shared memory where it fits.  A histogram of the logits' distance to the largest says which
// bins can hold the border of top_k (exactly) or of top_p (the bins' masses to a part in ten thousand); the few tokens
// of these bins are sorted by one CTA, against exact sums of what lies before them.  Where a bin holds more than kList
// tokens (thousands of equal logits) the border is found by bisection of the rank.
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

constexpr int kList = 1024;           // tokens that are sorted: one to a thread
constexpr int kBins = 2048;           // two to a thread
constexpr int kMargins = 4;

struct SampleSmem {
  double exp2[kTable];
  u64 part[32], slot[2];
  u64 list[kList];
  uint32_t count[kBins];
  int size;                           // of the list
  int first[1 + 2 * kMargins];        // the first bin at which a sum over the bins passes a value
  u64 cut;
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

// 2^42 exp((l - top) rate / log2(e)).  2^y = 2^k 2^(j/64) 2^f, |f| <= 1/128: the Taylor polynomial of degree 5 is within
// (ln 2 / 128)^6 / 720 = 4e-17 of 2^f.
struct Weights {
  const double* table;
  float top;                          // the largest logit
  double rate;                        // log2(e) / temperature
  __device__ double operator()(float l) const {
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
    return q * table[i & (kTable - 1)] * scale;
  }
};
__device__ __forceinline__ u64 units(double w) { return (u64)__double_as_longlong(w + 4503599627370496.0) & ((1ull << 52) - 1); }

struct Settings {
  double temperature, top_p, least;   // least: 2^42 min_p
  long long top_k;
  float u;
  __device__ Settings(const SampleParams& p, int row) {
    temperature = p.temperature != nullptr ? p.temperature[row] : p.temperature0;
    top_p = p.top_p != nullptr ? p.top_p[row] : p.top_p0;
    least = fmin(fmax(p.min_p != nullptr ? p.min_p[row] : p.min_p0, 0.0), 1.0) * (double)kOne;
    top_k = p.top_k != nullptr ? p.top_k[row] : p.top_k0;
    u = p.u[row];
  }
  // the weight that the kept tokens have to reach
  __device__ u64 reach(u64 total) const {
    if (!(top_p < 1.0)) return ~0ull;
    const double t = ceil(top_p * (double)total);
    return t > 1.0 ? (u64)t : 1;
  }
  __device__ u64 draw(u64 total) const {
    const double t = (double)u * (double)total;
    return t > 0.0 ? min((u64)t, total - 1) : 0;
  }
};

__device__ __forceinline__ float load_logit(const SampleParams& p, int row, int i) {
  return p.bf16 ? ssm::to_f32(static_cast<const __nv_bfloat16*>(p.logits)[row * p.stride + i])
                : static_cast<const float*>(p.logits)[row * p.stride + i];
}
// The rank of a logit as it came: a NaN above all.
__device__ __forceinline__ u64 raw_key(float l, int i) { return l != l ? ~0ull : rank_key(l, i); }
__device__ __forceinline__ int key_token(u64 key) { return (int)(0xffffffffu - (uint32_t)key); }
// Neither a token nor a choice: no logit above -inf, a NaN, a NaN temperature.
__device__ __forceinline__ bool no_token(u64 best, double temperature) {
  return best == ~0ull || key_logit(best) == -__int_as_float(0x7f800000) || temperature != temperature;
}

// ---- a CTA's threads, a value each ------------------------------------------------------------------
// The sum up to each thread, and of all.
__device__ __forceinline__ u64 block_scan(u64 v, u64* part, u64* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int m = 1; m < 32; m *= 2) {
    const u64 up = __shfl_up_sync(0xffffffffu, v, m);
    if (lane >= m) v += up;
  }
  if (lane == 31) part[warp] = v;
  __syncthreads();
  u64 w = lane < warps ? part[lane] : 0;
#pragma unroll
  for (int m = 1; m < 32; m *= 2) {
    const u64 up = __shfl_up_sync(0xffffffffu, w, m);
    if (lane >= m) w += up;
  }
  const u64 before = __shfl_sync(0xffffffffu, w, max(0, warp - 1));
  *total = __shfl_sync(0xffffffffu, w, 31);
  __syncthreads();
  return warp > 0 ? v + before : v;
}
__device__ __forceinline__ u64 block_max(u64 v, u64* part) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int m = 16; m >= 1; m /= 2) v = max(v, __shfl_xor_sync(0xffffffffu, v, m));
  if (lane == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = lane < (int)(blockDim.x >> 5) ? part[lane] : 0;
#pragma unroll
  for (int m = 16; m >= 1; m /= 2) v = max(v, __shfl_xor_sync(0xffffffffu, v, m));
  __syncthreads();
  return v;
}
// The first n threads' values (n a power of two, 32 or more), largest first: a bitonic network, by shuffles within a warp.
__device__ __forceinline__ u64 block_sort(u64 v, u64* buf, int n) {
  for (int size = 2; size <= n; size *= 2)
    for (int stride = size / 2; stride >= 1; stride /= 2) {
      u64 other;
      if (stride >= 32) {
        buf[threadIdx.x] = v;
        __syncthreads();
        other = buf[threadIdx.x ^ stride];
        __syncthreads();
      } else {
        other = __shfl_xor_sync(0xffffffffu, v, stride);
      }
      const bool larger = ((threadIdx.x & size) == 0) == ((threadIdx.x & stride) == 0);
      if (threadIdx.x < n) v = larger ? max(v, other) : min(v, other);
    }
  return v;
}

// Up to kList tokens, one to a thread.
__global__ void __launch_bounds__(kList) sample_few(const __grid_constant__ SampleParams p) {
  __shared__ u64 part[32], buf[kList];
  __shared__ double table[kTable];
  const int row = (int)blockIdx.x, i = threadIdx.x;
  const Settings set(p, row);
  if (i < kTable) table[i] = exp2((double)i / kTable);
  const float l = i < p.V ? load_logit(p, row, i) : 0.0f;
  u64 key = i < p.V ? raw_key(l, i) : 0;
  const u64 best = block_max(key, part);
  const bool none = no_token(best, set.temperature);
  if (none || !(set.temperature > 0.0)) {
    if (i == 0) p.token[row] = none ? -1 : key_token(best);
    return;
  }
  const Weights weight{table, key_logit(best), 1.4426950408889634 / set.temperature};
  u64 total, w = 0;
  const bool top_k = set.top_k > 0 && set.top_k < p.V;
  if (top_k || set.top_p < 1.0) {
    key = block_sort(key, buf, (int)blockDim.x);
    const double exact = key != 0 && (!top_k || i < set.top_k) ? weight(key_logit(key)) : 0.0;
    w = units(exact);
    const u64 run = block_scan(w, part, &total);
    if (key != 0) buf[key_token(key)] = run - w < set.reach(total) && exact >= set.least ? w : 0;
    __syncthreads();
    w = i < p.V ? buf[i] : 0;
  } else if (i < p.V) {
    const double exact = weight(l);
    w = exact >= set.least ? units(exact) : 0;
  }
  const u64 run = block_scan(w, part, &total), target = set.draw(total);
  if (run > target && run - w <= target) p.token[row] = i;
}

// ---- a cluster's threads, many tokens each --------------------------------------------------------------
struct Sampler {
  const SampleParams& p;
  SampleSmem& s;
  cg::cluster_group cluster;
  int row, ctas, lane, warp, base, first, last, turn;
  Weights weight;
  float bin_rate;                     // bins to a logit

  __device__ Sampler(const SampleParams& p_, SampleSmem& s_) : p(p_), s(s_), cluster(cg::this_cluster()), turn(0) {
    ctas = (int)cluster.num_blocks();
    row = (int)blockIdx.x / ctas;
    lane = threadIdx.x & 31;
    warp = threadIdx.x >> 5;
    // a warp's tokens are neighbours, so that warps in order are tokens in order
    base = min(p.V, (int)cluster.block_rank() * p.slice);
    const int end = min(p.V, base + p.slice), per = ((end - base + 31) / 32 + 31) & ~31;
    first = min(end, base + warp * per);
    last = min(end, first + per);
    weight.table = s.exp2;
  }
  __device__ float logit(int i) const { return p.cached ? s.logits[i - base] : load_logit(p, row, i); }

  // The sum (or maximum) over the cluster's threads, for all of them.
  template <bool MAX>
  __device__ u64 join(u64 v) {
    auto f = [](u64 a, u64 b) { return MAX ? max(a, b) : a + b; };
#pragma unroll
    for (int m = 16; m >= 1; m /= 2) v = f(v, __shfl_xor_sync(0xffffffffu, v, m));
    if (lane == 0) s.part[warp] = v;
    __syncthreads();
    v = s.part[lane];
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
  __device__ void sync() {
    if (ctas == 1) __syncthreads();
    else cluster.sync();
  }

  // The bin of a logit by its distance to the largest; kBins: so far below that its weight is zero.
  __device__ int bin(float l) const {
    const float z = l == weight.top ? 0.0f : (weight.top - l) * bin_rate;
    return z < (float)kBins ? (int)z : kBins;
  }

  // How many tokens (or what weight) rank at least as high as both keys.
  template <bool MASS>
  __device__ u64 above(u64 cut, u64 key) {
    u64 n = 0;
    const u64 least = max(cut, key);
    for (int i = first + lane; i < last; i += 32) {
      const float l = logit(i);
      if (rank_key(l, i) >= least) n += MASS ? units(weight(l)) : 1;
    }
    return join<false>(n);
  }
  // The key of the token, by rank, at which the count (or weight) of those that rank at least as high as `cut`
  // reaches `target`; one that has all of them where it does not.
  template <bool MASS>
  __device__ u64 bisect(u64 cut, u64 target) {
    u64 lo = 0, hi = ~0ull;               // above(lo) >= target (or lo = 0), above(hi + 1) < target
    while (lo < hi) {
      const u64 mid = lo + (hi - lo) / 2 + 1;
      if (above<MASS>(cut, mid) >= target) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  }

  // Every bin's count over the cluster, in registers: bins 2 t and 2 t + 1 of thread t.
  __device__ void count_bins(uint32_t (&n)[2]) {
    for (int b = threadIdx.x; b < kBins; b += kList) s.count[b] = 0;
    if (threadIdx.x < 1 + 2 * kMargins) s.first[threadIdx.x] = kBins - 1;
    if (threadIdx.x == 0) s.size = 0;
    __syncthreads();
    for (int i = first + lane; i < last; i += 32) {
      const int b = bin(logit(i));
      if (b < kBins) atomicAdd(&s.count[b], 1u);
    }
    sync();
    n[0] = n[1] = 0;
    for (int r = 0; r < ctas; ++r) {
      const uint2 c = *reinterpret_cast<const uint2*>(cluster.map_shared_rank(s.count, r) + 2 * threadIdx.x);
      n[0] += c.x;
      n[1] += c.y;
    }
  }
  // The tokens of bins lo .. hi that rank at least as high as `cut`, in the first CTA's list (in any order); f(l, bin,
  // in) is called for each token.
  template <typename F>
  __device__ void gather(int lo, int hi, u64 cut, F f) {
    int* size = cluster.map_shared_rank(&s.size, 0);
    u64* list = cluster.map_shared_rank(s.list, 0);
    for (int i = first + lane; i < last; i += 32) {
      const float l = logit(i);
      const int b = bin(l);
      const u64 key = rank_key(l, i);
      if (b >= lo && b <= hi && key >= cut) {
        const int at = atomicAdd(size, 1);
        if (at < kList) list[at] = key;
      }
      f(l, b, key);
    }
  }
  // This thread's token of the first CTA's list, largest first (0: none); for all CTAs of the cluster to call.
  __device__ u64 sorted() {
    sync();                               // the list is written
    const int n = min(s.size, kList);     // 0 but in the first CTA
    int pow2 = 32;
    while (pow2 < n) pow2 *= 2;
    const u64 key = (int)threadIdx.x < n ? s.list[threadIdx.x] : 0;
    __syncthreads();
    return block_sort(key, s.list, pow2);
  }
};

__global__ void __launch_bounds__(kList) sample_many(const __grid_constant__ SampleParams p) {
  extern __shared__ __align__(16) unsigned char raw[];
  SampleSmem& s = *reinterpret_cast<SampleSmem*>(raw);
  Sampler a(p, s);
  const Settings set(p, a.row);
  const int t = threadIdx.x;
  const bool leader = a.cluster.block_rank() == 0;
  if (t < kTable) s.exp2[t] = exp2((double)t / kTable);
  u64 best = 0, worst = 0;                                // the lowest as the highest of the negated
  const float inf = __int_as_float(0x7f800000);
#pragma unroll 4
  for (int i = a.first + a.lane; i < a.last; i += 32) {
    const float l = load_logit(p, a.row, i);
    if (p.cached) s.logits[i - a.base] = l;
    best = max(best, raw_key(l, i));
    if (l != -inf) worst = max(worst, raw_key(-l, i));
  }
  best = a.join<true>(best);
  const bool none = no_token(best, set.temperature);
  if (none || !(set.temperature > 0.0)) {                 // the same for the whole cluster
    if (t == 0 && leader) p.token[a.row] = none ? -1 : key_token(best);
    a.sync();                                             // peers read this CTA's slots until here
    return;
  }
  a.weight.top = key_logit(best);
  a.weight.rate = 1.4426950408889634 / set.temperature;
  const bool top_k = set.top_k > 0 && set.top_k < p.V, top_p = set.top_p < 1.0;
  u64 cut = 0;
  if (top_k || top_p) {
    worst = a.join<true>(worst);
    // 31 temperatures below the largest a weight is zero
    const float range = fminf(31.0f * (float)set.temperature, a.weight.top + key_logit(worst));
    a.bin_rate = ((float)kBins - 0.01f) / range;
    uint32_t n[2];
    a.count_bins(n);
    u64 all;
    const u64 count1 = block_scan((u64)n[0] + n[1], s.part, &all), count0 = count1 - n[1];   // up to bin 2 t + 1, 2 t
    int last = kBins - 1;                                 // the bin of the top_k-th token
    u64 listed = all;                                     // tokens up to it
    if (top_k && (u64)set.top_k < all) {
      const u64 k = (u64)set.top_k;
      if (count1 >= k && count1 - n[0] - n[1] < k) s.first[0] = count0 >= k ? 2 * t : 2 * t + 1;
      __syncthreads();
      last = s.first[0];
      if (last >> 1 == t) s.slot[a.turn] = last & 1 ? count1 : count0;
      __syncthreads();
      listed = s.slot[a.turn];
      __syncthreads();
    }
    if (listed <= kList) {                                // what is kept of the top_k: all in the list
      a.gather(0, last, 0, [](float, int, u64) {});
      u64 key = a.sorted();
      a.sync();
      if (!leader) return;
      const long long k = top_k ? set.top_k : p.V;
      const double exact = key != 0 && t < k ? a.weight(key_logit(key)) : 0.0;
      u64 w = units(exact), total;
      u64 run = block_scan(w, s.part, &total);
      // by index: the token in the high half, its logit's order in the low one
      key = w != 0 && run - w < set.reach(total) && exact >= set.least ? key << 32 | key >> 32 : 0;
      int pow2 = 32;
      while (pow2 < (int)listed) pow2 *= 2;
      key = block_sort(key, s.list, pow2);
      w = key != 0 ? units(a.weight(key_logit(key << 32 | key >> 32))) : 0;
      run = block_scan(w, s.part, &total);
      const u64 target = set.draw(total);
      if (run > target && run - w <= target) p.token[a.row] = key_token(key >> 32);
      return;
    }
    if (top_k && (u64)set.top_k < all) {                  // the border of top_k lies in bin `last`
      if (last >> 1 == t) s.slot[a.turn] = last & 1 ? count0 : count0 - n[0];
      __syncthreads();
      const u64 before = s.slot[a.turn];
      __syncthreads();
      if (listed - before > kList) {
        cut = a.bisect<false>(0, (u64)set.top_k);
      } else {
        a.gather(last, last, 0, [](float, int, u64) {});
        const u64 key = a.sorted();
        if (leader && t == (int)((u64)set.top_k - before) - 1) s.cut = key;
        a.sync();
        cut = *a.cluster.map_shared_rank(&s.cut, 0);
        if (t == 0) s.size = 0;
        a.sync();
      }
    }
    if (top_p) {
      // the bins' masses, about: as many weights as it has tokens, from its middle
      const float step = range / ((float)kBins - 0.01f) / (float)set.temperature;
      const int b = 2 * t;
      const float m0 = b <= last ? (float)n[0] * __expf(-step * ((float)b + 0.5f)) : 0.0f;
      const float m1 = b < last ? (float)n[1] * __expf(-step * ((float)b + 1.5f)) : 0.0f;
      u64 mass;
      const u64 unit0 = (u64)(m0 * 16777216.0f), unit1 = (u64)(m1 * 16777216.0f);
      const u64 run1 = block_scan(unit0 + unit1, s.part, &mass), run0 = run1 - unit1, run = run0 - unit0;
      // the bins between (top_p - margin) and (top_p + margin) of the mass, for the widest margin whose tokens fit
      const double margins[kMargins] = {0.008, 0.001, 0.0001, 0.0};
      auto mark = [&](int at, u64 value) {                // the first bin at which the sum is above `value`
        if (run <= value && run1 > value) s.first[at] = run0 > value ? b : b + 1;
      };
#pragma unroll
      for (int i = 0; i < kMargins; ++i) {
        mark(1 + 2 * i, (u64)fmax(0.0, (set.top_p - margins[i]) * (double)mass));
        mark(2 + 2 * i, (u64)fmax(0.0, (set.top_p + margins[i]) * (double)mass));
      }
      // tokens up to every bin; the histogram's own counts are not needed again
      a.sync();
      s.count[b] = (uint32_t)count0;
      s.count[b + 1] = (uint32_t)count1;
      __syncthreads();
      int lo = 0, hi = 0;
      bool fits = false;
      for (int i = 0; i < kMargins && !fits; ++i) {
        lo = s.first[1 + 2 * i];
        hi = min(last, s.first[2 + 2 * i]);
        fits = s.count[hi] - (lo > 0 ? s.count[lo - 1] : 0) <= kList;
      }
      u64 total = 0, before = 0;
      if (fits) {
        a.gather(lo, hi, cut, [&](float l, int bin, u64 key) {
          if (bin >= kBins || key < cut) return;
          const u64 w = units(a.weight(l));
          total += w;
          if (bin < lo) before += w;
        });
        const u64 key = a.sorted();
        total = a.join<false>(total);
        before = a.join<false>(before);
        const u64 reach = set.reach(total), w = key != 0 ? units(a.weight(key_logit(key))) : 0;
        u64 sum;
        const u64 upto = before + block_scan(w, s.part, &sum);
        // the border is in the list: the last token that the sum before it leaves short
        if (t == 0) s.cut = 0;
        __syncthreads();
        if (leader && key != 0 && upto - w < reach && upto >= reach) s.cut = key;
        a.sync();
        const u64 found = *a.cluster.map_shared_rank(&s.cut, 0);
        fits = found != 0;
        if (fits) cut = found;
      } else {
        total = a.above<true>(cut, 0);
      }
      if (!fits) cut = max(cut, a.bisect<true>(cut, set.reach(total)));
    }
  }
  auto kept = [&](int i) -> u64 {
    const float l = a.logit(i);
    if (rank_key(l, i) < cut) return 0;
    const double w = a.weight(l);
    return w >= set.least ? units(w) : 0;
  };
  u64 sum = 0;
  for (int i = a.first + a.lane; i < a.last; i += 32) sum += kept(i);
  // what the warps and CTAs before have
#pragma unroll
  for (int m = 16; m >= 1; m /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, m);
  u64 cta;
  u64 before = block_scan(a.lane == 31 ? sum : 0, s.part, &cta), total = cta;
  before = __shfl_sync(0xffffffffu, before, 31) - sum;
  if (a.ctas > 1) {
    if (t == 0) s.slot[a.turn] = cta;
    a.cluster.sync();
    total = 0;
    for (int r = 0; r < a.ctas; ++r) {
      const u64 v = *a.cluster.map_shared_rank(&s.slot[a.turn], r);
      if (r < (int)a.cluster.block_rank()) before += v;
      total += v;
    }
  }
  const u64 target = set.draw(total);
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
  a.sync();
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
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (V <= kList) {
    int threads = kTable;                                  // a power of two: one token to a thread
    while (threads < V) threads *= 2;
    sample_few<<<(unsigned)B, threads, 0, st>>>(p);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? SSM_OK : fail(SSM_ERR_CUDA, "sample_tokens launch failed (error %lld)", (long long)e);
  }
  // CTAs to a row: what keeps the slices in shared memory, and more where few rows leave SMs idle
  int ctas = 1;
  while (ctas < 8 && V > (int64_t)ctas * kCached) ctas *= 2;
  while (ctas < 8 && V >= (int64_t)ctas * 8192 && B * ctas * 2 <= 148) ctas *= 2;
  p.slice = (int)((V + ctas - 1) / ctas);
  p.cached = p.slice <= kCached;
  ssm::ctas_per_sm<sample_many>(kList, sizeof(SampleSmem) + kCached * sizeof(float));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(B * ctas));
  cfg.blockDim = dim3(kList);
  cfg.dynamicSmemBytes = sizeof(SampleSmem) + (p.cached ? p.slice * sizeof(float) : 0);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_many, p);
  return e == cudaSuccess ? SSM_OK : fail(SSM_ERR_CUDA, "sample_tokens launch failed (error %lld)", (long long)e);
}
