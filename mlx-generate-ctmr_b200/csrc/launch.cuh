// Kernel launches with programmatic dependent launch (PDL).
//
// Every kernel of this library is launched with the stream attribute that lets
// it start while the previous kernel in the stream is still finishing, and
// every kernel calls griddep_wait() before it touches global memory (the
// persistent conv kernels after their shared-memory / TMEM set-up). The wait
// returns once the preceding grid has completed and its writes are visible, so
// the ordering of a plain launch is kept while the launch latency and the
// set-up overlap the predecessor's tail. Each kernel signals
// griddep_launch_dependents() right away (one that takes tensor memory once its
// block holds it): its successor may then be scheduled as soon as this grid's
// last blocks are resident.
//
// One pair of kernels goes further: adapter_linear's product kernels, behind
// their inner products, read x, the weight, the offsets and the bias before the
// wait, and may write rows of y that no adapter meets. That is in order because
// the inner kernel waits before it signals (so everything older is complete when
// the product starts), reads x alone of these and writes none, and because every
// block of the product waits before it ends.
//
// Inside a CUDA-graph capture the attribute becomes a programmatic edge.
// CTMR_DISABLE_PDL=1 turns it off.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstdlib>
#include <utility>

namespace ctmr {

__device__ __forceinline__ void griddep_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void griddep_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;"); }

// Streaming multiprocessors of the current device: the unit every grid-size plan of this
// library is measured in (148 on a B200). Queried once per device.
inline int device_sm_count() {
  static std::atomic<int> cached[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0) return 148;
  if (dev < 64) {
    const int hit = cached[dev].load(std::memory_order_relaxed);
    if (hit > 0) return hit;
  }
  int n = 0;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) return 148;
  if (dev < 64) cached[dev].store(n, std::memory_order_relaxed);
  return n;
}

inline bool pdl_enabled() {
  static const bool on = std::getenv("CTMR_DISABLE_PDL") == nullptr;
  return on;
}

// A kernel's opt-in to more than 48 KB of shared memory (and, where asked, to clusters of 16), requested
// once per device: the request takes longer than a small kernel's launch. One static object per kernel.
class SharedMemoryGrant {
 public:
  template <typename Kernel>
  cudaError_t ensure(Kernel kern, size_t bytes, bool large_clusters = false) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 64 && (done_.load(std::memory_order_acquire) >> dev & 1)) return cudaSuccess;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    if (e == cudaSuccess && large_clusters)
      e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess && dev < 64) done_.fetch_or(1ull << dev, std::memory_order_release);
    return e;
  }

 private:
  std::atomic<unsigned long long> done_{0};
};

template <typename... KArgs, typename... Args>
cudaError_t launch_kernel(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                          Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
}

}  // namespace ctmr
