// ssm_launch.cuh — host side of launches with dynamic shared memory.
#pragma once

#include <cuda_runtime.h>

#include <atomic>

namespace ssm {

// Raises Kern's shared memory limit to `smem` on the current device and returns how many of its CTAs fit on an SM
// (0 after an error, which the launch then reports).  Asked of the driver once per kernel and device: the two
// calls cost more host time than a small launch.
template <auto Kern>
int ctas_per_sm(int threads, size_t smem) {
  static std::atomic<int> known[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (dev < 64)
    if (const int n = known[dev].load(std::memory_order_relaxed)) return n;
  int n = 0;
  if (cudaFuncSetAttribute(Kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) return 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, Kern, threads, smem) != cudaSuccess) return 0;
  if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
  return n;
}

// The same for a kernel that is launched with different numbers of threads (whole warps, up to 32) and `smem` bytes for
// these; `most`: the largest of all its launches, to which the limit is set every time (two host threads may be here at once).
template <auto Kern>
int ctas_per_sm_threads(int threads, size_t smem, size_t most) {
  static std::atomic<int> known[64][33];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (dev < 64)
    if (const int n = known[dev][threads / 32].load(std::memory_order_relaxed)) return n;
  int n = 0;
  if (cudaFuncSetAttribute(Kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most) != cudaSuccess) return 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, Kern, threads, smem) != cudaSuccess) return 0;
  if (dev < 64) known[dev][threads / 32].store(n, std::memory_order_relaxed);
  return n;
}

}  // namespace ssm
