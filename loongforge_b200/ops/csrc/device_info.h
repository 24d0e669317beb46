// What launchers ask about the current device, asked of the driver once per device: such a call costs as much as a launch.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>
#include <atomic>

namespace lf {

// Multiprocessors of the current device; those of a B200 where it cannot be asked.
inline int sm_count() {
  constexpr int kDevices = 64, kB200 = 148;
  static std::atomic<int> known[kDevices];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0) return kB200;
  if (dev < kDevices && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return kB200;
  if (dev < kDevices) known[dev].store(n, std::memory_order_relaxed);
  return n;
}

// Lets `kernel` have that much shared memory; `done` is the kernel's own.
template <typename K>
bool allow_smem(K kernel, size_t bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_relaxed) & bit)) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)) != cudaSuccess) return false;
  if (dev < 64) done.fetch_or(bit, std::memory_order_relaxed);
  return true;
}

}  // namespace lf
