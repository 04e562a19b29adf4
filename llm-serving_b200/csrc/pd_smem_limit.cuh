// pd_smem_limit.cuh -- a kernel's dynamic shared memory limit, raised once per device.
#pragma once

#include <cuda_runtime.h>

#include <atomic>

namespace pd {

// Raises a kernel's dynamic shared memory limit on the current device, once. The limit is the kernel's, not
// the call's, so that first calls of two host threads set the same value whatever they need themselves.
constexpr int SMEM_MAX_DEVICES = 64;
using SmemRaised = std::atomic<bool>[SMEM_MAX_DEVICES];
template <typename Kernel>
cudaError_t raise_smem_limit(Kernel fn, int bytes, SmemRaised& raised) {
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess || (dev < SMEM_MAX_DEVICES && raised[dev].load(std::memory_order_acquire))) return err;
  err = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (err == cudaSuccess && dev < SMEM_MAX_DEVICES) raised[dev].store(true, std::memory_order_release);
  return err;
}

}  // namespace pd
