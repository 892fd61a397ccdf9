// Launches of the 16-bit cache's kernels.
//
// Every kernel is launched programmatically: its CTAs may become resident while the stream's previous kernel still runs, and
// each waits (after_previous) for that kernel's end before it touches global memory.  No thread block returns before that, so a
// kernel never ends before the one in front of it, and a stream's order holds.  It hides 2 to 4 us of a launch (decode of 32 x
// 1028 visible tokens: 38.6 -> 34.3 us together with the batched join).  The eviction's copies do not invite the next kernel
// early (let_next_start): a next selection's clusters that wait beside them cost 5 us.
#pragma once
#include <cuda_runtime.h>

#include <atomic>

#include "k16_common.cuh"

namespace k16 {

FR_DEVI void let_next_start() { asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory"); }
FR_DEVI void after_previous() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }

// What a launch needs to know about the current device, looked up once per device: its SMs, and that a kernel may use its
// dynamic shared memory (the attribute belongs to the kernel on one device).
constexpr int MAX_DEVICES = 64;
inline cudaError_t device_sms(int& dev, int& sms) {
  static std::atomic<int> known[MAX_DEVICES];
  if (cudaError_t e = cudaGetDevice(&dev)) return e;
  sms = dev < MAX_DEVICES ? known[dev].load(std::memory_order_relaxed) : 0;
  if (sms > 0) return cudaSuccess;
  const cudaError_t e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e == cudaSuccess && dev < MAX_DEVICES) known[dev].store(sms, std::memory_order_relaxed);
  return e;
}
template <class K> cudaError_t allow_smem(K kernel, int bytes, int dev, std::atomic<bool> (&done)[MAX_DEVICES]) {
  if (dev < MAX_DEVICES && done[dev].load(std::memory_order_relaxed)) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < MAX_DEVICES) done[dev].store(true, std::memory_order_relaxed);
  return e;
}

template <class... Ts>
cudaError_t launch(void (*k)(Ts...), unsigned grid, unsigned threads, size_t smem, int cluster, cudaStream_t st, const Ts&... args) {
  cudaLaunchAttribute at[2];
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3(grid);
  c.blockDim = dim3(threads);
  c.dynamicSmemBytes = smem;
  c.stream = st;
  c.attrs = at;
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  c.numAttrs = 1;
  if (cluster > 0) {
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    c.numAttrs = 2;
  }
  return cudaLaunchKernelEx(&c, k, args...);
}

}  // namespace k16
