// A kernel's shared memory settings, made once for each device.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace dn {

// Allows KERNEL `bytes` of dynamic shared memory, with the SM's whole split for
// it: blocks of two kernels stay on one SM only under the same split. The two
// calls cost the host about a microsecond each, so a device's are remembered
// (devices past 63 are set every time); setting them twice is harmless.
template <auto KERNEL>
inline cudaError_t allow_smem(int bytes) {
  static std::atomic<uint64_t> known{0};
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return e;
  const uint64_t bit = dev >= 0 && dev < 64 ? (uint64_t)1 << dev : 0;
  if ((known.load(std::memory_order_relaxed) & bit) != 0) return cudaSuccess;
  if (cudaError_t e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
      e != cudaSuccess)
    return e;
  if (cudaError_t e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributePreferredSharedMemoryCarveout,
                                           cudaSharedmemCarveoutMaxShared);
      e != cudaSuccess)
    return e;
  known.fetch_or(bit, std::memory_order_relaxed);
  return cudaSuccess;
}

}  // namespace dn
