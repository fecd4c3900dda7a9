// Host helpers of the plaintext operators (no context).
#pragma once
#include <atomic>

#include "b2f_internal.h"

namespace b2f {

// The current device and its SM count (asked once per device).
inline int current_device(int *dev, int *sms) {
  static std::atomic<int> known[64];
  B2F_CUDA(cudaGetDevice(dev));
  const int slot = *dev & 63;
  int n = *dev < 64 ? known[slot].load(std::memory_order_relaxed) : 0;
  if (!n) {
    B2F_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, *dev));
    if (*dev < 64) known[slot].store(n, std::memory_order_relaxed);
  }
  *sms = n;
  return B2F_OK;
}

// Lets a kernel take `bytes` of dynamic shared memory on device dev; `done` is the
// kernel's own record of the devices where it may.
template <class K>
int allow_shared(K kernel, int bytes, int dev, std::atomic<uint64_t> &done) {
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return B2F_OK;
  B2F_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  done.fetch_or(bit, std::memory_order_relaxed);
  return B2F_OK;
}

}  // namespace b2f
