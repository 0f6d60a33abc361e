// What the translation units of libfbmm.so share on the host side: the calling thread's error
// message, the per-device check and the tensor-map encoder. Defined in fbmm_api.cu.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

namespace fbmm_host {

// Stores the message fbmm_last_error() returns; gives `code` back.
int fail(int code, const char* fmt, ...);

// FBMM_OK and the SM count when the current device is one this library runs on.
int device_sms(int* sms);

// SM count of the current device, or the B200's where no device can be asked (the workspace queries work on
// a machine without one).
int sms_or_default();

// 3-D tiled tensor map (dims, strides in bytes of dims 1 and 2, box), 128-byte or no swizzle, from
// the cache of recent maps where it is there.
int tensor_map_3d(CUtensorMap* map, CUtensorMapDataType type, const void* base, const cuuint64_t dims[3],
                  const cuuint64_t strides[2], const cuuint32_t box[3], bool swizzle128);

// Reads and clears the status word of the microscaled kernels (fbmm_mx_api.cu).
int mx_status(unsigned int* bits);

}  // namespace fbmm_host

#define FBMM_HOST_CUDA(call)                                                                                       \
  do {                                                                                                             \
    cudaError_t e_ = (call);                                                                                       \
    if (e_ != cudaSuccess) return fbmm_host::fail(FBMM_ERR_CUDA, "%s: %s", #call, cudaGetErrorString(e_));         \
  } while (0)
