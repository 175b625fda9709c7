// ssm_sample.cu — the next token of every row of logits, from a given uniform number.
//
// Of w = exp((l - max) / temperature): the top_k largest are kept; of these, largest first, as many as it takes for their
// sum to reach top_p of all of theirs; of these what is at least min_p.  The token is the first, by index, where the running
// sum of the kept weights passes u times their sum.  Equal logits rank by index.
//
// A token must not depend on how sums are split, nor change when a sum's rounding does: weights are whole numbers in
// units of 2^-42, formed in double, and every sum is a 64-bit whole number, exact in any order (up to 2^20 tokens).  A weight
// is cut down by less than 2^-42 of the largest; what is less than that is never drawn.
//
// Up to kFew tokens: a thread each, sorted by rank in registers (a byte of one sequence: 7 us, most of it the launch).
// More: a cluster of up to eight CTAs shares a row, a slice of tokens each, kept in shared memory where two CTAs to an SM have
// the room.  A histogram of the logits' distance to the largest says which bins can hold the border of top_k (exactly) or
// of top_p (the bins' masses to a part in ten thousand); the few tokens of these bins are sorted by one CTA, against exact
// sums of what lies before them.  Where the bins' masses mislead, the exact sum at the list's edge says where to look next; where
// a bin holds more than kList tokens (hundreds of equal logits) a pass over the row takes eleven bits of the border's rank.
//
// 256 x 131072 fp32 by top-p: 138 us, 0.4 GB of DRAM in three passes, whose loads are four ahead in slots of shared memory.  The
// 108 SMs that have two rows decide (263 thousand clocks: maximum 38, histogram 64, list and sums 115, all else 45); a row
// that has its SM alone takes 218, so what bounds a row is the latency of its passes' chains (a load, the table, a weight's double
// arithmetic), and only the fifth that the second row adds is issue slots, 55 % of which are used over the GPU.  By temperature
// alone 72 us, by top-k 75.  64 x 50257 bf16 with all rules: 18 us,
// the barriers of passes of 1 to 3 us each.  Bisection of the rank, the first form, took 6690 and 518 us.
#include <cooperative_groups.h>

#include <algorithm>
#include <cstdio>
#include <type_traits>

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
  int wide;                           // rows start where four logits are one load
  int cached;                         // its logits are kept in shared memory
};

constexpr int kBits = 42;
constexpr u64 kOne = 1ull << kBits;
constexpr int kTable = 1024;          // steps of the table of 2^x; 2^10
constexpr int kFew = 1024;            // tokens that one CTA takes, one to a thread
constexpr int kThreads = 512;         // of a CTA that shares a row: two of them to an SM, so that one waits while one works
constexpr int kWarps = kThreads / 32;
constexpr int kList = kThreads;       // tokens that are sorted: one to a thread
constexpr int kPer = 4, kBins = kPer * kThreads;
constexpr int kMargins = 4;
constexpr int kDepth = 4;              // loads of a thread on their way, where a row is not kept

// What a gather adds up: nothing, all weights and those before a bin, those of some bins.
enum Adds { kNothing, kAll, kSome };

struct SampleSmem {
  double exp2[kTable];
  u64 part[32], part2[kWarps], slot[2], slot2[2];
  u64 list[kList];
  u64 kept[kWarps];                   // by warp: the weight of its kept tokens
  uint32_t count[kBins], upto[kBins];
  int size;                           // of the list
  int first[1 + 2 * kMargins];        // the first bin at which a sum over the bins passes a value
  u64 cut, rest;                      // rest: what the drawn token's place is short of where its warp's tokens start
  int owner;                          // that warp
  int half;                           // see Sampler::form
  alignas(16) float logits[4];        // the slice, or kDepth slots of 16 bytes to a thread
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
__device__ __forceinline__ int key_token(u64 key) { return (int)(0xffffffffu - (uint32_t)key); }

// ln 2, its square by 2, its cube by 6: from constant memory an operand of the instruction, not two moves before it.
constexpr double kLn2 = 0.69314718055994531;
__constant__ double kTaylor[3] = {kLn2, kLn2 * kLn2 / 2, kLn2 * kLn2 * kLn2 / 6};

// A weight in whole units: 2^42 2^y cut to a whole number, y = (l - top) rate, for finite top and l <= top.  2^y = 2^k 2^(j/1024)
// 2^r, |r| <= 2^-11: the Taylor polynomial of degree 3 is within (ln 2 / 2048)^4 / 24 = 6e-16 of 2^r.  y is held above -60, where
// the weight is zero, by its high word: of two negative numbers the larger has the smaller one.
struct Weights {
  static constexpr double kRaised = 4503599627370496.0;
  const double* table;                // 2^(42 + j / 1024), its high word less j 2^10: adding 1024 y 2^10 adds k to the exponent
  double top, rate;                   // the largest logit; log2(e) / temperature, held within 1e-290 .. 1e290
  __device__ void set(float top_, double temperature) {
    top = top_;
    rate = fmin(fmax(1.4426950408889634 / temperature, 1e-290), 1e290);
  }
  static __device__ double entry(int j) {
    const double v = exp2((double)j / kTable + kBits);
    return __hiloint2double(__double2hiint(v) - (j << 10), __double2loint(v));
  }
  // The sum and the weight, cut to a whole number by the addition itself: the sum is a whole number of 2^52 up to 2^53, where
  // doubles are a unit apart, and rounding down is the same whatever it is added to.  A thread starts its sum at kRaised
  // and has up to 2^10 tokens.  The passes over whole rows are bound by the instructions they issue: this takes two off.
  __device__ __forceinline__ double add(float l, double sum) const {
    constexpr double kShift = 6755399441055744.0 / kTable;   // 1.5 2^52 / 1024: y is rounded to 1024ths
    const double raw = ((double)l - top) * rate;
    const double y = __hiloint2double((int)min((uint32_t)__double2hiint(raw), 0xc04e0000u), __double2loint(raw));      // -60
    const double t = y + kShift;
    const int i = __double2loint(t);                       // 1024 y, rounded
    const double r = y - (t - kShift);
    const double q = fma(r, fma(r, fma(r, kTaylor[2], kTaylor[1]), kTaylor[0]), 1.0);
    const double step = table[i & (kTable - 1)];
    const double scaled = __hiloint2double(__double2hiint(step) + i * kTable, __double2loint(step));
    return __fma_rd(scaled, q, sum);
  }
  __device__ __forceinline__ u64 operator()(float l) const {
    return (u64)__double_as_longlong(add(l, kRaised)) & ((1ull << 52) - 1);
  }
  static __device__ u64 whole(double sum) { return (u64)(sum - kRaised); }
};

// Whether a token ranks at least as high as one with this key.
struct Border {
  float l;
  int i;
  __device__ explicit Border(u64 key)
      : l(key != 0 ? key_logit(key) : -__builtin_huge_valf()), i(key != 0 ? key_token(key) : 0x7fffffff) {}
  __device__ __forceinline__ bool operator()(float v, int at) const { return v > l || (v == l && at <= i); }
};

struct Settings {
  double temperature, top_p;
  u64 least;                          // min_p
  long long top_k;
  float u;
  __device__ Settings(const SampleParams& p, int row) {
    temperature = p.temperature != nullptr ? p.temperature[row] : p.temperature0;
    top_p = p.top_p != nullptr ? p.top_p[row] : p.top_p0;
    least = (u64)ceil(fmin(fmax(p.min_p != nullptr ? p.min_p[row] : p.min_p0, 0.0), 1.0) * (double)kOne);
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

// The rank of a logit as it came: a NaN above all.
__device__ __forceinline__ u64 raw_key(float l, int i) { return l != l ? ~0ull : rank_key(l, i); }
// Neither a token nor a choice: no logit above -inf, a NaN, a NaN temperature.
__device__ __forceinline__ bool no_token(u64 best, double temperature) {
  return best == ~0ull || key_logit(best) == -__int_as_float(0x7f800000) || temperature != temperature;
}

// The larger one, or NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
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

// Up to kFew tokens, one to a thread.
template <typename T>
__global__ void __launch_bounds__(kFew) sample_few(const __grid_constant__ SampleParams p) {
  __shared__ u64 part[32], buf[kFew];
  ssm::pdl_launch_dependents();
  ssm::pdl_wait();
  const int row = (int)blockIdx.x, i = threadIdx.x;
  const Settings set(p, row);
  const float l = i < p.V ? ssm::to_f32(static_cast<const T*>(p.logits)[row * p.stride + i]) : 0.0f;
  u64 key = i < p.V ? raw_key(l, i) : 0;
  const u64 best = block_max(key, part);
  const bool none = no_token(best, set.temperature);
  if (none || !(set.temperature > 0.0)) {
    if (i == 0) p.token[row] = none ? -1 : key_token(best);
    return;
  }
  const double top = key_logit(best), rate = 1.4426950408889634 / set.temperature;
  auto weight = [&](float v) {                            // as in Weights, by the library's function: no table to make
    const double y = ((double)v - top) * rate;
    return v == key_logit(best) ? kOne : y > -60.0 ? (u64)__double2ll_rd(exp2(y) * (double)kOne) : 0;
  };
  u64 total, w = 0;
  const bool top_k = set.top_k > 0 && set.top_k < p.V;
  if (top_k || set.top_p < 1.0) {
    key = block_sort(key, buf, (int)blockDim.x);
    w = key != 0 && (!top_k || i < set.top_k) ? weight(key_logit(key)) : 0;
    const u64 run = block_scan(w, part, &total);
    if (key != 0) buf[key_token(key)] = run - w < set.reach(total) && w >= set.least ? w : 0;
    __syncthreads();
    w = i < p.V ? buf[i] : 0;
  } else if (i < p.V) {
    w = weight(l);
    if (w < set.least) w = 0;
  }
  const u64 run = block_scan(w, part, &total), target = set.draw(total);
  if (run > target && run - w <= target) p.token[row] = i;
}

// ---- a cluster's threads, many tokens each --------------------------------------------------------------
template <typename T>
struct Sampler {
  const SampleParams& p;
  SampleSmem& s;
  cg::cluster_group cluster;
  const T* logits;                    // of the row
  int row, ctas, lane, warp, base, per, first, last, turn;
  Weights weight;
  float top, bin_rate;                // the largest logit; bins to a logit
  bool formed;                        // the passes work on other values than the logits

  __device__ Sampler(const SampleParams& p_, SampleSmem& s_) : p(p_), s(s_), cluster(cg::this_cluster()), turn(0), formed(false) {
    ctas = (int)cluster.num_blocks();
    row = (int)blockIdx.x / ctas;
    logits = static_cast<const T*>(p.logits) + row * p.stride;
    lane = threadIdx.x & 31;
    warp = threadIdx.x >> 5;
    // a warp's tokens are neighbours, so that warps in order are tokens in order; four to a lane and step
    base = min(p.V, (int)cluster.block_rank() * p.slice);
    const int end = min(p.V, base + p.slice);
    per = ((end - base + kWarps - 1) / kWarps + 127) & ~127;
    first = min(end, base + warp * per);
    last = min(end, first + per);
    weight.table = s.exp2;
  }
  // In a row with infinite logits these alone count: 0, and -inf the others.  Where a float does not hold how far logits are apart and
  // the temperature is so high that it matters, halves of both (exact but for logits below 2^-125, which are then one to any weight).
  __device__ __forceinline__ float form(float l) const {
    constexpr float kInf = __builtin_huge_valf();
    return s.half ? 0.5f * l : l == kInf ? 0.0f : -kInf;
  }
  // Four logits from i on; -inf past the warp's last.
  __device__ void load(int i, float (&l)[4]) const {
    constexpr float kInf = __builtin_huge_valf();
    if (p.wide && i + 4 <= last) {
      ssm::load4(logits + i, l);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) l[j] = i + j < last ? ssm::to_f32(logits[i + j]) : -kInf;
    }
    if (formed) {
#pragma unroll
      for (int j = 0; j < 4; ++j) l[j] = form(l[j]);
    }
  }
  __device__ void keep(int i, const float (&l)[4]) {
    *reinterpret_cast<float4*>(s.logits + (i - base)) = make_float4(l[0], l[1], l[2], l[3]);
  }
  // f(i, l[4]) for this lane's tokens
  template <typename F>
  __device__ __forceinline__ void each(F f) {
    if (p.cached) {
      for (int i = first + 4 * lane; i < last; i += 128) {
        float l[4];
        ssm::load4(s.logits + (i - base), l);
        f(i, l);
      }
    } else if (p.wide && !formed) {       // from L2 or memory: the next ones on their way to this thread's slots
      constexpr uint32_t kStep = kThreads * 16, kRing = kDepth * kStep;
      const uint32_t ring = ssm::smem_u32(s.logits) + threadIdx.x * 16;
      const T* from = logits + first + 4 * lane;
      const int steps = (last - first) >> 7;              // that are whole for the warp
      auto fetch = [&](int step, const T* src, uint32_t at) {
        if (step < steps)
          asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(ring + at), "l"(src), "n"(4 * sizeof(T)) : "memory");
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
#pragma unroll
      for (int d = 0; d < kDepth; ++d) fetch(d, from + 128 * d, d * kStep);
      int i = first + 4 * lane;
      uint32_t at = 0;
      for (int step = 0; step < steps; ++step) {
        float l[4];
        asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
        ssm::load4(reinterpret_cast<const T*>(reinterpret_cast<const char*>(s.logits) + threadIdx.x * 16 + at), l);
        f(i, l);
        fetch(step + kDepth, from + 128 * kDepth, at);
        from += 128;
        i += 128;
        at = (at + kStep) & (kRing - 1);
      }
      if (i < last) {
        float l[4];
        load(i, l);
        f(i, l);
      }
    } else {
      for (int i = first + 4 * lane; i < last; i += 128) {
        float l[4];
        load(i, l);
        f(i, l);
      }
    }
  }

  // The sum (or maximum, or HALVES: the maxima of the two halves) over the cluster's threads, for all of them.
  template <bool MAX, bool HALVES = false>
  __device__ u64 join(u64 v) {
    auto f = [](u64 a, u64 b) {
      if (HALVES) return (u64)max((uint32_t)(a >> 32), (uint32_t)(b >> 32)) << 32 | max((uint32_t)a, (uint32_t)b);
      return MAX ? max(a, b) : a + b;
    };
    auto of_warp = [&](u64 v) {
      if constexpr (HALVES) {
        return (u64)__reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32)) << 32 | __reduce_max_sync(0xffffffffu, (uint32_t)v);
      } else {
#pragma unroll
        for (int m = 16; m >= 1; m /= 2) v = f(v, __shfl_xor_sync(0xffffffffu, v, m));
        return v;
      }
    };
    v = of_warp(v);
    if (lane == 0) s.part[warp] = v;
    __syncthreads();
    v = of_warp(lane < kWarps ? s.part[lane] : 0);
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

  __device__ __forceinline__ float distance(float l) const { return (top - l) * bin_rate; }
  // The bin of a logit by its distance to the largest; kBins: so far below that its weight is zero.
  __device__ int bin(float l) const {
    const float z = distance(l);
    return z < (float)kBins ? (int)z : kBins;
  }

  // The largest key of a logit that is `b` bins or more from the largest: a search over the floats, by every thread.
  __device__ u64 highest_key(int b) const {
    if (b == 0) return ~0ull;
    uint32_t lo = 0x007fffffu, hi = (uint32_t)(rank_key(top, 0) >> 32);     // -inf is that far, the largest is not
    while (hi - lo > 1) {
      const uint32_t mid = lo + (hi - lo) / 2;
      if (distance(key_logit((u64)mid << 32)) >= (float)b) lo = mid;
      else hi = mid;
    }
    return (u64)lo << 32 | 0xffffffffu;
  }
  // The key lo <= key <= hi of the token, by rank, with which the count (or weight) of those from hi on, and `before`, reaches
  // `target`.  A pass takes eleven bits of the range: a bin to each part of it, exact sums in the bins.  False: all of them do not
  // reach it; lo is the key, `before` their sum.
  template <bool MASS>
  __device__ bool search(u64& lo, u64 hi, u64& before, u64 target) {
    using Bin = std::conditional_t<MASS, u64, uint32_t>;
    Bin* bins = reinterpret_cast<Bin*>(s.count);          // sums take the place of `upto` too
    while (lo < hi) {
      const int shift = max(0, 64 - __clzll((long long)(hi - lo)) - 11);
      sync();                                             // the bins are no longer read
      for (int b = threadIdx.x; b < kBins; b += kThreads) bins[b] = 0;
      if (threadIdx.x == 0) s.first[0] = -1;
      __syncthreads();
      each([&](int i, const float (&l)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const u64 key = rank_key(l[j], i + j);
          if (i + j < last && key >= lo && key <= hi) {
            if constexpr (MASS) atomicAdd(&bins[(hi - key) >> shift], weight(l[j]));
            else atomicAdd(&bins[(hi - key) >> shift], 1u);
          }
        }
      });
      sync();
      u64 n[kPer] = {}, mine = 0, all;
      for (int r = 0; r < ctas; ++r) {
        const Bin* of = cluster.map_shared_rank(bins, r) + kPer * threadIdx.x;
#pragma unroll
        for (int i = 0; i < kPer; ++i) n[i] += of[i];
      }
#pragma unroll
      for (int i = 0; i < kPer; ++i) mine += n[i];
      u64 upto = before + block_scan(mine, s.part, &all) - mine;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        if (upto < target && upto + n[i] >= target) {
          s.first[0] = kPer * threadIdx.x + i;
          s.rest = upto;
        }
        upto += n[i];
      }
      __syncthreads();
      const int bin = s.first[0];
      if (bin < 0) {
        before += all;
        return false;
      }
      before = s.rest;
      hi -= (u64)bin << shift;
      const u64 span = (1ull << shift) - 1;
      if (hi - lo > span) lo = hi - span;
    }
    return true;
  }

  // Every bin's count over the cluster, in registers: kPer bins to a thread.
  __device__ void count_bins(uint32_t (&n)[kPer]) {
    for (int b = threadIdx.x; b < kBins; b += kThreads) s.count[b] = 0;
    if (threadIdx.x < 1 + 2 * kMargins) s.first[threadIdx.x] = kBins - 1;
    if (threadIdx.x == 0) s.size = 0;
    __syncthreads();
    each([&](int, const float (&l)[4]) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int b = bin(l[j]);
        if (b < kBins) atomicAdd(&s.count[b], 1u);
      }
    });
    sync();
#pragma unroll
    for (int i = 0; i < kPer; ++i) n[i] = 0;
    for (int r = 0; r < ctas; ++r) {
      const uint4 c = *reinterpret_cast<const uint4*>(cluster.map_shared_rank(s.count, r) + kPer * threadIdx.x);
      n[0] += c.x;
      n[1] += c.y;
      n[2] += c.z;
      n[3] += c.w;
    }
  }
  // The tokens of bins lo .. hi that rank at least as high as `cut` to the first CTA's list (in any order).  kAll: of the tokens
  // that rank so, the weight of all and of those in bins below lo.  kSome: of those in bins from .. to - 1.
  template <Adds ADDS>
  __device__ void gather(int lo, int hi, u64 cut, u64& total, u64& before, int from = 0, int to = 0) {
    int* size = cluster.map_shared_rank(&s.size, 0);
    u64* list = cluster.map_shared_rank(s.list, 0);
    const float begin = (float)lo, end = (float)(hi + 1), some = (float)from, others = (float)to;
    const Border border(cut);
    double all = Weights::kRaised, higher = Weights::kRaised;
    auto body = [&](int i, const float (&l)[4], auto cuts) {
      bool here[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float z = distance(l[j]);
        const bool in = !cuts || border(l[j], i + j);
        if constexpr (ADDS == kAll) {
          const float v = in ? l[j] : -__builtin_huge_valf();
          all = weight.add(v, all);
          if (z < begin) higher = weight.add(v, higher);
        } else if constexpr (ADDS == kSome) {
          if (in && z >= some && z < others) higher = weight.add(l[j], higher);
        }
        here[j] = z >= begin && z < end && in;
      }
      if (here[0] || here[1] || here[2] || here[3]) {     // one branch to four tokens, after their weights
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (!here[j]) continue;
          const int at = atomicAdd(size, 1);
          if (at < kList) list[at] = rank_key(l[j], i + j);
        }
      }
    };
    if (cut != 0) each([&](int i, const float (&l)[4]) { body(i, l, std::true_type()); });
    else each([&](int i, const float (&l)[4]) { body(i, l, std::false_type()); });
    total = Weights::whole(all);
    before = Weights::whole(higher);
  }
  // x and y summed over the cluster, once the list is written: one barrier of the cluster for both.
  __device__ void sums(u64& x, u64& y) {
#pragma unroll
    for (int m = 16; m >= 1; m /= 2) {
      x += __shfl_xor_sync(0xffffffffu, x, m);
      y += __shfl_xor_sync(0xffffffffu, y, m);
    }
    if (lane == 0) s.part[warp] = x, s.part2[warp] = y;
    __syncthreads();
    if (warp == 0) {
      x = lane < kWarps ? s.part[lane] : 0;
      y = lane < kWarps ? s.part2[lane] : 0;
#pragma unroll
      for (int m = 16; m >= 1; m /= 2) {
        x += __shfl_xor_sync(0xffffffffu, x, m);
        y += __shfl_xor_sync(0xffffffffu, y, m);
      }
      if (lane == 0) s.slot[turn] = x, s.slot2[turn] = y;
    }
    sync();                               // the list and the sums are written
    x = y = 0;
    for (int r = 0; r < ctas; ++r) {
      x += *cluster.map_shared_rank(&s.slot[turn], r);
      y += *cluster.map_shared_rank(&s.slot2[turn], r);
    }
    turn ^= 1;
  }
  // This thread's token of the first CTA's list, which is written, largest first (0: none; in the other CTAs all).
  __device__ u64 sorted() {
    const int n = min(s.size, kList);
    const u64 key = (int)threadIdx.x < n ? s.list[threadIdx.x] : 0;
    if (n > 128) {
      int pow2 = 256;
      while (pow2 < n) pow2 *= 2;
      __syncthreads();
      return block_sort(key, s.list, pow2);
    }
    // few: every token's rank by comparing it with all
    int rank = 0;
    if (key != 0)
      for (int i = 0; i < n; ++i) rank += s.list[i] > key;
    __syncthreads();
    if (key != 0) s.list[rank] = key;
    __syncthreads();
    return (int)threadIdx.x < n ? s.list[threadIdx.x] : 0;
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_many(const __grid_constant__ SampleParams p) {
  extern __shared__ __align__(16) unsigned char raw[];
  SampleSmem& s = *reinterpret_cast<SampleSmem*>(raw);
  const int t = threadIdx.x;
  for (int i = t; i < kTable; i += kThreads) s.exp2[i] = Weights::entry(i);
  ssm::pdl_launch_dependents();
  ssm::pdl_wait();
  Sampler<T> a(p, s);
  const Settings set(p, a.row);
  const bool leader = a.cluster.block_rank() == 0;
  constexpr float kInf = __builtin_huge_valf();
  float high = -kInf, low = kInf;                         // of the logits above -inf
#pragma unroll 4
  for (int i = a.first + 4 * a.lane; i < a.last; i += 128) {
    float l[4];
    a.load(i, l);
    if (p.cached) a.keep(i, l);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      high = max_nan(high, l[j]);
      low = fminf(low, l[j] > -kInf ? l[j] : kInf);
    }
  }
  // both in one: the largest, and the smallest as the largest of the negated
  const u64 ends = a.template join<true, true>(high != high ? ~0ull : (rank_key(high, 0) >> 32) << 32 | rank_key(-low, 0) >> 32);
  const bool none = no_token(ends, set.temperature);
  a.top = key_logit(ends);
  if (none || !(set.temperature > 0.0)) {                 // the same for the whole cluster
    u64 best = 0;
    if (!none)
      a.each([&](int i, const float (&l)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (i + j < a.last) best = max(best, rank_key(l[j], i + j));
      });
    best = a.template join<true>(best);
    if (t == 0 && leader) p.token[a.row] = none ? -1 : key_token(best);
    a.sync();                                             // peers read this CTA's slots until here
    return;
  }
  float spread = a.top + key_logit(ends << 32);           // between the largest and the smallest above -inf
  float heat = (float)set.temperature;                    // held as a float, which is enough for the bins
  double temperature = set.temperature;
  if (a.top == kInf || (spread == kInf && 31.0f * heat == kInf)) {
    const bool half = a.top < kInf;
    s.half = half;                                        // by every thread, before it reads it
    a.formed = true;
    spread = half ? 0.5f * a.top + 0.5f * key_logit(ends << 32) : 0.0f;
    a.top = half ? 0.5f * a.top : 0.0f;
    if (half) temperature *= 0.5;
    heat = (float)temperature;
    for (int i = a.first + 4 * a.lane; p.cached && i < a.last; i += 128) {
      float l[4];
      a.load(i, l);
      a.keep(i, l);
    }
  }
  a.weight.set(a.top, temperature);
  const bool top_k = set.top_k > 0 && set.top_k < p.V, top_p = set.top_p < 1.0;
  u64 cut = 0;
  bool summed = false;                                    // s.kept is known
  if (top_k || top_p) {
    // 31 temperatures below the largest a weight is zero
    const float range = fminf(31.0f * heat, spread);
    a.bin_rate = fminf(((float)kBins - 0.01f) / range, 3e38f);
    uint32_t n[kPer];
    a.count_bins(n);
    u64 all, run = block_scan((u64)n[0] + n[1] + n[2] + n[3], s.part, &all) - n[0] - n[1] - n[2] - n[3];
    const int b0 = kPer * t;                              // this thread's first bin
    int last = kBins - 1;                                 // the bin of the top_k-th token
    const bool borders = top_k && (u64)set.top_k < all;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (borders && run < (u64)set.top_k && run + n[i] >= (u64)set.top_k) s.first[0] = b0 + i;
      s.upto[b0 + i] = (uint32_t)(run += n[i]);
    }
    __syncthreads();
    if (borders) last = s.first[0];
    const int listed = (int)s.upto[last];                 // tokens up to it
    if (listed <= kList) {                                // what is kept of the top_k: all in the list
      u64 none0, none1;
      a.template gather<kNothing>(0, last, 0, none0, none1);
      a.sync();
      if (!leader) return;                                // nobody reads this CTA's memory any more
      u64 key = a.sorted();
      const long long k = top_k ? set.top_k : p.V;
      u64 w = key != 0 && t < k ? a.weight(key_logit(key)) : 0, total;
      run = block_scan(w, s.part, &total);
      // by index: the token in the high half, its logit's order in the low one
      key = w != 0 && run - w < set.reach(total) && w >= set.least ? key << 32 | key >> 32 : 0;
      int pow2 = 32;
      while (pow2 < listed) pow2 *= 2;
      key = block_sort(key, s.list, pow2);
      w = key != 0 ? a.weight(key_logit(key << 32 | key >> 32)) : 0;
      run = block_scan(w, s.part, &total);
      const u64 target = set.draw(total);
      if (run > target && run - w <= target) p.token[a.row] = key_token(key >> 32);
      return;
    }
    if (borders) {                                        // the border of top_k lies in bin `last`
      const int before = last > 0 ? (int)s.upto[last - 1] : 0;
      if (listed - before > kList) {
        cut = a.highest_key(last + 1) + 1;
        u64 upto = before;
        a.template search<false>(cut, a.highest_key(last), upto, (u64)set.top_k);
      } else {
        u64 none0, none1;
        a.template gather<kNothing>(last, last, 0, none0, none1);
        a.sync();
        const u64 key = a.sorted();
        if (leader && t == (int)set.top_k - before - 1) s.cut = key;
        a.sync();
        cut = *a.cluster.map_shared_rank(&s.cut, 0);
        if (t == 0) s.size = 0;
        a.sync();
      }
    }
    if (top_p) {
      // The masses of this thread's bins, about: as many weights as a bin has tokens, from its middle, in units of 2^-24.  They
      // are made anew when they are needed again, which is rare: held over the pass in between they cost it registers.
      const float step = range / ((float)kBins - 0.01f) / heat;
      auto masses = [&](u64 (&unit)[kPer], u64& upto) {   // upto: before the first of the thread's bins.  The mass of all.
        u64 mine = 0, mass;
        uint32_t seen = b0 > 0 ? s.upto[b0 - 1] : 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const uint32_t now = borders && b0 + i == last ? (uint32_t)set.top_k : s.upto[b0 + i];
          unit[i] = b0 + i <= last ? (u64)((float)(now - seen) * __expf(-step * ((float)(b0 + i) + 0.5f)) * 16777216.0f) : 0;
          mine += unit[i];
          seen = now;
        }
        upto = block_scan(mine, s.part, &mass) - mine;
        return mass;
      };
      u64 unit[kPer], upto;
      const u64 mass = masses(unit, upto);
      // the first bin at which the sum is above (top_p - margin), and (top_p + margin), of the mass
      const double margins[kMargins] = {0.008, 0.001, 0.0001, 0.0};
#pragma unroll
      for (int i = 0; i < 2 * kMargins; ++i) {
        const double share = set.top_p + (i & 1 ? margins[i / 2] : -margins[i / 2]);
        const u64 value = (u64)fmax(0.0, share * (double)mass);
        u64 at = upto;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          if (at <= value && at + unit[j] > value) s.first[1 + i] = b0 + j;
          at += unit[j];
        }
      }
      __syncthreads();
      // the widest margin with few tokens, else the widest with as many as fit, else the widest of all
      auto tokens = [&](int lo, int hi) { return (int)(s.upto[hi] - (lo > 0 ? s.upto[lo - 1] : 0)); };
      int lo = 0, hi = 0;
      bool fits = false;
      for (int most = kList / 4; most <= kList && !fits; most *= 4)
        for (int i = 0; i < kMargins - (most < kList) && !fits; ++i) {
          lo = s.first[1 + 2 * i];
          hi = min(last, s.first[2 + 2 * i]);
          fits = tokens(lo, hi) <= most;
        }
      if (!fits) {
        lo = s.first[1];
        hi = min(last, s.first[2]);
      }
      u64 total, before;                                  // before: the weight of what lies before bin lo
      a.template gather<kAll>(lo, hi, cut, total, before);
      auto of_warp = [](u64 v) {
#pragma unroll
        for (int m = 16; m >= 1; m /= 2) v += __shfl_xor_sync(0xffffffffu, v, m);
        return v;
      };
      u64 mine = of_warp(before);
      if (a.lane == 0) s.kept[a.warp] = mine;
      a.sums(total, before);
      const u64 reach = set.reach(total);
      bool found = false;
      // where the border is if it is not found: between these bins, with so much before them
      int from = lo, to = hi;
      u64 start = before;
      for (int turn = 0; fits; ++turn) {
        u64 key = a.sorted();
        const u64 w = key != 0 ? a.weight(key_logit(key)) : 0;
        u64 sum;
        const u64 run = before + block_scan(w, s.part, &sum);
        // the border is in the list: the last token that the sum before it leaves short
        if (t == 0) {
          s.cut = s.size = 0;
          s.rest = sum;
        }
        s.list[t] = key;
        __syncthreads();
        if (leader && key != 0 && run - w < reach && run >= reach) s.cut = key;
        a.sync();
        const u64 border = *a.cluster.map_shared_rank(&s.cut, 0);
        found = border != 0;
        if (found) {
          cut = border;
          key = a.cluster.map_shared_rank(s.list, 0)[t];
          const int at = key_token(key) - a.base;
          if (key >= cut && at >= 0 && at < p.slice) atomicAdd(&s.kept[at / a.per], a.weight(key_logit(key)));
          summed = a.weight(key_logit(cut)) >= set.least;  // min_p cuts nothing off
        }
        __syncthreads();                                  // s.kept is written; s.first and s.part2 are no longer read
        if (found || turn == 1) break;
        // It is off by a known weight from an edge of the list: where the bins' masses say, from there on.
        const bool after = reach > before;
        const u64 edge = after ? before + *a.cluster.map_shared_rank(&s.rest, 0) : before;
        from = after ? hi + 1 : 0;
        to = after ? last : lo - 1;
        start = after ? edge : 0;
        const int old = lo, at = after ? hi + 1 : lo;
        masses(unit, upto);
        u64 e = upto;
        if (t < 4) s.first[1 + t] = last;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          if (b0 + j == at) s.part2[0] = e;
          e += unit[j];
        }
        __syncthreads();
        if (from > to) break;                             // no such bin
        const long long off = ((long long)reach - (long long)edge) >> (kBits - 24), slack = (off < 0 ? -off : off) / 32 + 8;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const long long value = max(0ll, (long long)s.part2[0] + off + (i == 0 ? -slack : i == 1 ? slack : 0));
          long long e2 = (long long)upto;
#pragma unroll
          for (int j = 0; j < kPer; ++j) {
            if (e2 <= value && e2 + (long long)unit[j] > value) s.first[1 + i] = b0 + j;
            e2 += (long long)unit[j];
          }
        }
        __syncthreads();
        fits = false;
        for (int i = 0; i < 4 && !fits; i += 2) {
          lo = min(max(s.first[1 + i], from), to);
          hi = max(min(s.first[2 + i], to), lo);
          fits = tokens(lo, hi) <= kList;
        }
        if (!fits) break;
        u64 none0;
        a.template gather<kSome>(lo, hi, cut, none0, mine, min(lo, old), max(lo, old));
        u64 part = mine, none1 = 0;
        mine = of_warp(mine);
        if (a.lane == 0) s.kept[a.warp] += after ? mine : 0 - mine;
        a.sums(part, none1);
        before += after ? part : 0 - part;
      }
      if (!found) {
        u64 lowest = max(cut, a.highest_key(to + 1) + 1), highest = a.highest_key(from);
        if (reach <= start) {
          highest = ~0ull;
          lowest = max(cut, a.highest_key(from) + 1);
          start = 0;
        }
        u64 key = lowest;
        if (!a.template search<true>(key, highest, start, reach) && lowest > cut) {
          key = cut;
          a.template search<true>(key, lowest - 1, start, reach);
        }
        cut = key;
      }
    }
  }
  const Border border(cut);
  u64 sum = 0;
  if (summed) {
    sum = s.kept[a.warp];
  } else {
    double kept = Weights::kRaised;                                    // past the warp's last token l is -inf, its weight zero
    if (cut == 0 && set.least == 0) {
      a.each([&](int, const float (&l)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) kept = a.weight.add(l[j], kept);
      });
    } else {
      const double least = (double)set.least;
      a.each([&](int i, const float (&l)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const double next = a.weight.add(l[j], kept);
          if (border(l[j], i + j) && next - kept >= least) kept = next;
        }
      });
    }
    sum = Weights::whole(kept);
#pragma unroll
    for (int m = 16; m >= 1; m /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, m);
  }
  // what the warps and CTAs before have
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
  // the warp whose tokens hold the drawn one; its CTA goes over them together
  const u64 target = set.draw(total);
  if (t == 0) s.owner = -1;
  __syncthreads();
  if (a.lane == 0 && before <= target && target < before + sum) {
    s.owner = a.warp;
    s.rest = target - before;
  }
  __syncthreads();
  if (s.owner >= 0) {
    const int begin = a.base + s.owner * a.per, end = min(min(p.V, a.base + p.slice), begin + a.per);
    u64 rest = s.rest;
    for (int at = begin; at < end; at += 4 * kThreads) {  // four tokens to a thread
      const int i = at + 4 * t;
      u64 w[4], own = 0, all;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float l = -kInf;
        if (i + j < end) {
          l = p.cached ? s.logits[i + j - a.base] : ssm::to_f32(a.logits[i + j]);
          if (a.formed && !p.cached) l = a.form(l);
        }
        w[j] = a.weight(l);
        if (!border(l, i + j) || w[j] < set.least) w[j] = 0;
        own += w[j];
      }
      u64 run = block_scan(own, s.part, &all) - own;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (run <= rest && run + w[j] > rest) p.token[a.row] = i + j;
        run += w[j];
      }
      if (rest < all) break;
      rest -= all;
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
constexpr int kCached = 19 * 1024;    // logits that each of two CTAs on an SM keeps (76 KB); more are read again

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
  if (V <= kFew) {
    int threads = 64;                                      // a power of two: one token to a thread
    while (threads < V) threads *= 2;
    const cudaError_t e = ssm::launch_pdl(p.bf16 ? sample_few<__nv_bfloat16> : sample_few<float>, (unsigned)B, threads, 0, st, p);
    return e == cudaSuccess ? SSM_OK : fail(SSM_ERR_CUDA, "sample_tokens launch failed (error %lld)", (long long)e);
  }
  // CTAs to a row: as many as run at once, and so many that a thread has up to 2^10 tokens (Weights::add).  A cluster's barriers
  // cost a row as much as its passes (256 x 131072 by top-p: 300 us with eight CTAs to a row, 158 with one).
  int ctas = 1;
  while (ctas < 8 && V >= (int64_t)ctas * 4096 && (B * ctas * 2 <= 296 || V > (int64_t)ctas << 19)) ctas *= 2;
  p.slice = (int)((V + ctas - 1) / ctas + 3) & ~3;
  p.cached = p.slice <= kCached;
  const int unit = p.bf16 ? 8 : 16;                        // bytes of four logits
  p.wide = reinterpret_cast<uintptr_t>(p.logits) % unit == 0 && p.stride % 4 == 0;
  const size_t most = sizeof(SampleSmem) + kCached * sizeof(float);
  if (p.bf16) ssm::ctas_per_sm<sample_many<__nv_bfloat16>>(kThreads, most);
  else ssm::ctas_per_sm<sample_many<float>>(kThreads, most);
  const size_t smem = sizeof(SampleSmem) + (p.cached ? p.slice * sizeof(float) : kDepth * kThreads * sizeof(uint4));
  const auto kern = p.bf16 ? sample_many<__nv_bfloat16> : sample_many<float>;
  const cudaError_t e = ssm::launch_pdl_cluster(kern, (unsigned)(B * ctas), kThreads, (unsigned)ctas, smem, st, p);
  return e == cudaSuccess ? SSM_OK : fail(SSM_ERR_CUDA, "sample_tokens launch failed (error %lld)", (long long)e);
}
