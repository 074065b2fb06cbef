// Host side of kernel launches.
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

#include <atomic>

namespace moe {

// Lets a kernel have `bytes` of dynamic LDS on the current device.  The runtime keeps
// that per device, so it is asked for once on each (`done`, one per kernel: a bit for
// each device).
inline hipError_t allow_lds(const void *kernel, int bytes, std::atomic<uint64_t> *done) {
  int device = 0;
  hipError_t e = hipGetDevice(&device);
  if (e != hipSuccess) return e;
  const uint64_t bit = device < 64 ? 1ull << device : 0ull;
  if (done->load(std::memory_order_relaxed) & bit) return hipSuccess;
  e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == hipSuccess) done->fetch_or(bit, std::memory_order_relaxed);
  return e;
}

}  // namespace moe
