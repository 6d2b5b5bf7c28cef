// The current device's CU count, asked once per device, and what a launch can hold (host code).
#pragma once

#include <hip/hip_runtime.h>

#include <atomic>

namespace mote {

inline int device_cu_count() {
  constexpr int kMost = 64;
  static std::atomic<int> known[kMost];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMost) return 256;
  int cus = known[dev].load(std::memory_order_relaxed);
  if (cus > 0) return cus;
  if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0) return 256;
  known[dev].store(cus, std::memory_order_relaxed);
  return cus;
}

// whether a grid's first dimension of so many workgroups can be launched: below 2^32 threads
inline bool grid_fits(int64_t workgroups, int threads) { return workgroups * threads < (int64_t(1) << 32); }

}  // namespace mote
