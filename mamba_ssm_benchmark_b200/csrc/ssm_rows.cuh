// ssm_rows.cuh — a warp's part of a row of a (rows, channels) tensor, wherever the row starts.
#pragma once

#include "ssm_vec.cuh"

namespace ssm {

// 16 bytes into shared memory, asynchronously: the first n of them from src, zeros behind.
__device__ __forceinline__ void fetch_unit(void* dst, const void* src, int n) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(n) : "memory");
}
// A warp's part of a row: VEC values to a lane, 32 VEC in a row from value c0 on, in 16-byte units of shared memory.
// RAGGED: rows start anywhere and end anywhere; the units are those of memory that hold the values, a lane reads its own and
// the next one and shifts.  (Loads of a value or two at a time, at 16384 x 2047 bf16: 515 us; this way 100.)
// Values are float2 pairs: one instruction takes two.  Issue slots bound these kernels as much as memory does.
template <typename T, int VEC, bool RAGGED>
struct Slot {
  static constexpr int kLane = VEC * (int)sizeof(T), kUnits = kLane / 16, kWords = kLane / 4;
  static constexpr int kWarp = 32 * kLane + (RAGGED ? 16 : 0);          // bytes
  static_assert(kLane % 16 == 0, "whole units");
  static __device__ __forceinline__ int offset(const T* row, int c0) {
    return (int)(reinterpret_cast<uintptr_t>(row + c0) & 15);
  }
  // The warp's units of a row to `at`, which held zeros at first: what lies past the row's end stays zero.
  static __device__ __forceinline__ void fetch(unsigned char* at, const T* row, int c0, int C, int lane) {
    if constexpr (RAGGED) {
      // a unit that holds a value of the row lies in the row's allocation up to that value: allocations start at multiples of 16
      const int o = offset(row, c0);
      const char* from = reinterpret_cast<const char*>(row + c0) - o;
      const char* none = reinterpret_cast<const char*>(reinterpret_cast<uintptr_t>(row) & ~uintptr_t(15));
      const int bytes = c0 < C ? (C - c0) * (int)sizeof(T) + o : 0;            // from the first unit to the row's end
#pragma unroll
      for (int i = 0; i <= kUnits; ++i) {
        const int u = i * 32 + lane, n = min(16, bytes - 16 * u);
        if (i < kUnits || lane == 0) fetch_unit(at + 16 * u, n > 0 ? from + 16 * u : none, max(n, 0));
      }
    } else {
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int c = c0 + (i * 32 + lane) * (16 / (int)sizeof(T));
        if (c < C) fetch_unit(at + (i * 32 + lane) * 16, row + c, 16);
      }
    }
  }
  // two values to a word pair or word, and back
  static __device__ __forceinline__ void pack(const float2 (&v)[VEC / 2], uint32_t (&w)[kWords]) {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      if constexpr (sizeof(T) == 4) {
        w[2 * i] = __float_as_uint(v[i].x);
        w[2 * i + 1] = __float_as_uint(v[i].y);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[i].x, v[i].y);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
  }
  static __device__ __forceinline__ void unpack(const uint32_t* w, float2 (&v)[VEC / 2]) {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      if constexpr (sizeof(T) == 4)
        v[i] = make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
      else
        v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    }
  }
  // The lane's values, zeros past the row's end.
  static __device__ __forceinline__ void read(const unsigned char* at, const T* row, int c0, int lane, float2 (&v)[VEC / 2]) {
    constexpr int kHeld = kWords + (RAGGED ? 4 : 0);
    uint32_t w[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld / 4; ++i) {
      const uint4 q = *reinterpret_cast<const uint4*>(at + (lane * kUnits + i) * 16);
      w[4 * i] = q.x, w[4 * i + 1] = q.y, w[4 * i + 2] = q.z, w[4 * i + 3] = q.w;
    }
    if constexpr (RAGGED) to_front(w, offset(row, c0));
    unpack(w, v);
  }
  // words towards the front by o bytes
  static __device__ __forceinline__ void to_front(uint32_t (&w)[kWords + 4], int o) {
#pragma unroll
    for (int i = 0; i + 2 < kWords + 4; ++i) w[i] = o & 8 ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i + 3 < kWords + 4; ++i) w[i] = o & 4 ? w[i + 1] : w[i];
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) w[i] = o & 2 ? __byte_perm(w[i], w[i + 1], 0x5432) : w[i];
    }
  }
  // the lane's words to the row; all lanes of a warp call it
  static __device__ __forceinline__ void write(T* row, int c0, int C, int lane, const uint32_t (&own)[kWords]) {
    constexpr int kVals = 16 / (int)sizeof(T);             // to a unit
    const int n = C - c0;                                  // values of the row in this warp, and behind it
    if constexpr (!RAGGED) {
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int first = (lane * kUnits + i) * kVals;
        if (first < n)
          *reinterpret_cast<uint4*>(row + c0 + first) = make_uint4(own[4 * i], own[4 * i + 1], own[4 * i + 2], own[4 * i + 3]);
      }
    } else {
      const int o = offset(row, c0), before = o / (int)sizeof(T);
      uint32_t w[kWords + 4];                              // the lane before's last unit, then this one's
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __shfl_up_sync(0xffffffffu, own[kWords - 4 + i], 1);
#pragma unroll
      for (int i = 0; i < kWords; ++i) w[4 + i] = own[i];
      // towards the back by o bytes: w[4] becomes the first word of this lane's first unit of memory, whose front is the end
      // of the lane before
#pragma unroll
      for (int i = kWords + 3; i >= 2; --i) w[i] = o & 8 ? w[i - 2] : w[i];
#pragma unroll
      for (int i = kWords + 3; i >= 3; --i) w[i] = o & 4 ? w[i - 1] : w[i];
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = kWords + 3; i >= 4; --i) w[i] = o & 2 ? __byte_perm(w[i - 1], w[i], 0x5432) : w[i];
      }
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int first = (lane * kUnits + i) * kVals - before;        // the unit's first value, from c0 on
        T* to = row + c0 + first;
        if (first >= 0 && first + kVals <= n)
          *reinterpret_cast<uint4*>(to) = make_uint4(w[4 + 4 * i], w[5 + 4 * i], w[6 + 4 * i], w[7 + 4 * i]);
        else
          single(to, -first, n - first, &w[4 + 4 * i]);
      }
      // what the last lane's shift moved out: the end of its last unit
      if (lane == 31 && before > 0) single(row + c0 + 32 * VEC - kVals, kVals - before, n - 32 * VEC + kVals, &own[kWords - 4]);
    }
  }
  // Without shared memory (VEC a unit): the unit of a row's memory at this lane, and from it and the next lane's the lane's
  // words.  RAGGED: the last lane has no next one, 31 lanes have values (kTaken of them).
  static constexpr int kTaken = (RAGGED ? 31 : 32) * VEC;
  static __device__ __forceinline__ uint4 take(const T* row, int c0, int C, int lane) {
    static_assert(kUnits == 1, "a unit to a lane");
    uint4 q = make_uint4(0, 0, 0, 0);
    if constexpr (!RAGGED) {
      if (c0 + lane * VEC < C) q = *reinterpret_cast<const uint4*>(row + c0 + lane * VEC);
    } else {
      const int o = offset(row, c0), n = c0 < C ? (C - c0) * (int)sizeof(T) + o - 16 * lane : 0;      // bytes to the row's end
      const T* from = row + c0 - o / (int)sizeof(T) + lane * VEC;
      if (n >= 16) {
        q = *reinterpret_cast<const uint4*>(from);
      } else if (n > 0) {                                  // not past the row's end, where the allocation may end too
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          if (i * (int)sizeof(T) >= n) continue;
          if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(from[i]);
          else w[i / 2] |= (uint32_t)__bfloat16_as_ushort(from[i]) << (i & 1 ? 16 : 0);
        }
        q = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    return q;
  }
  static __device__ __forceinline__ void taken(const uint4& q, const T* row, int c0, uint32_t (&own)[kWords]) {
    if constexpr (!RAGGED) {
      own[0] = q.x, own[1] = q.y, own[2] = q.z, own[3] = q.w;
    } else {
      uint32_t w[kWords + 4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) w[4 + i] = __shfl_down_sync(0xffffffffu, w[i], 1);
      to_front(w, offset(row, c0));
#pragma unroll
      for (int i = 0; i < 4; ++i) own[i] = w[i];
    }
  }
  // values from .. to - 1 of a unit
  static __device__ __forceinline__ void single(T* unit, int from, int to, const uint32_t* w) {
#pragma unroll
    for (int i = 0; i < 16 / (int)sizeof(T); ++i) {
      if (i < from || i >= to) continue;
      if constexpr (sizeof(T) == 4)
        unit[i] = __uint_as_float(w[i]);
      else
        unit[i] = __ushort_as_bfloat16((unsigned short)(i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffff));
    }
  }
};

}  // namespace ssm
