// What launchers ask about the current device, asked of the driver once per device: such a call costs as much as a launch.
#pragma once
#include <cuda_runtime.h>
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

}  // namespace lf
