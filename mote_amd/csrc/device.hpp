// The current device's CU count, asked once per device (host code).
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

}  // namespace mote
