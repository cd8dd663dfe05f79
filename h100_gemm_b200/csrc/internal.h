// What the translation units of the library share on the host side (not part of the C ABI).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <cstdlib>

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

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Whether a launch may overlap the kernel before it in the stream (B200_GEMM_NO_PDL=1 turns that off).
inline int programmatic_launch() { return std::getenv("B200_GEMM_NO_PDL") ? 0 : 1; }

// A launch of a one-dimensional grid in stream order, in clusters, with the set-up overlapping the kernel before it: the
// kernel waits for that one to complete before it touches what it may write or still read.
struct Launch {
  cudaLaunchConfig_t config = {};
  cudaLaunchAttribute attr[2];
  Launch(long long grid, int threads, size_t smem, cudaStream_t stream, int cluster = 1) {
    config.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
    config.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = programmatic_launch();
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    config.attrs = attr;
    config.numAttrs = cluster > 1 ? 2 : 1;
  }
};

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
