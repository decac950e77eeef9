// What the launches of kernels share on the host.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <mutex>

#include "asterq_internal.h"

namespace asterq {

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// cuTensorMapEncodeTiled, without linking to the driver's library; null where it is not there.  It needs a current context,
// which a host thread has from its first call of the runtime that works on the device: this one, where the thread has made none.
inline EncodeTiled encode_tiled() {
  static thread_local bool bound = false;
  int dev = 0;
  if (!bound) bound = cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess;
  static const EncodeTiled fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
                   q == cudaDriverEntryPointSuccess
               ? reinterpret_cast<EncodeTiled>(ptr)
               : nullptr;
  }();
  return fn;
}

// A map of 16-bit values in boxes of 64 of the first dim (128 bytes, swizzled); strides in bytes, of the dims from the
// second on.
inline bool map_of_16bit(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
                         const cuuint32_t* box) {
  const cuuint32_t step[5] = {1u, 1u, 1u, 1u, 1u};
  const EncodeTiled fn = encode_tiled();
  return fn && fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, rank, const_cast<void*>(base), dims, strides, box, step,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Held while a call makes launches that hand records to each other in its workspace: host threads that share a stream, and with it
// a workspace, would otherwise put a launch of one call between those of another, which then joins the wrong records.
inline std::mutex& launch_lock() {
  static std::mutex lock;
  return lock;
}

// SMs of the current device and its ordinal; 0 where there is none
inline int current_sms(int* dev) {
  int n = 0;
  if (cudaGetDevice(dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, *dev) != cudaSuccess)
    return 0;
  return n;
}

}  // namespace asterq
