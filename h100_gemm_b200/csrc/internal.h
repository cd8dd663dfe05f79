// What the translation units of the library share on the host side (not part of the C ABI).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>

#include "../../include/b200_gemm.h"

namespace b200 {

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

struct DeviceInfo {
  int ordinal;
  int sm_count;
  int smem_optin;
  unsigned int* status;  // the device's four-word status block
  EncodeTiledFn encode;
};

// The current device's description (one-time set-up on first use); a b200_status code.
int device_info(DeviceInfo* out);

// Records a CUDA error for b200_gemm_last_cuda_error and returns B200_ERR_CUDA.
int cuda_failed(int error);

#define B200_TRY_CUDA(expr)                                                    \
  do {                                                                         \
    cudaError_t e__ = (expr);                                                  \
    if (e__ != cudaSuccess) {                                                  \
      (void)cudaGetLastError();                                                \
      return ::b200::cuda_failed(static_cast<int>(e__));                       \
    }                                                                          \
  } while (0)

// Lets a kernel use all of the device's shared memory; asked for once per device (`done`: the kernel's own flags).
template <typename Kernel>
int allow_shared_memory(const DeviceInfo& dev, Kernel kernel, std::atomic<bool> (&done)[64]) {
  if (!done[dev.ordinal].load(std::memory_order_acquire)) {
    B200_TRY_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, dev.smem_optin));
    done[dev.ordinal].store(true, std::memory_order_release);
  }
  return B200_OK;
}

}  // namespace b200
