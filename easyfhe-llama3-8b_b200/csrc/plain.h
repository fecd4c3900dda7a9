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

// Launches a kernel of a chain.  `chained`: it may start while the kernel before it
// in the stream still runs (programmatic dependent launch); every thread block of such
// a kernel, and of the one it follows, passes wait_for_previous before it touches what
// that one writes, so a kernel has ended only when all before it have.
template <class... P, class... A>
int launch_chained(void (*kernel)(P...), dim3 grid, dim3 block, size_t shared, int cluster,
                   bool chained, cudaStream_t s, A... args) {
  cudaLaunchConfig_t c{};
  c.gridDim = grid;
  c.blockDim = block;
  c.dynamicSmemBytes = shared;
  c.stream = s;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (cluster > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = cluster;
    at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
    ++n;
  }
  if (chained) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  c.attrs = at;
  c.numAttrs = n;
  B2F_CUDA(cudaLaunchKernelEx(&c, kernel, static_cast<P>(args)...));
  note_launch();
  return B2F_OK;
}
#ifdef __CUDACC__
// the kernel after this one in the stream may start
__device__ __forceinline__ void let_next_start() {
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
}
// all that the kernel before this one wrote is there
__device__ __forceinline__ void wait_for_previous() {
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
}
#endif

}  // namespace b2f
