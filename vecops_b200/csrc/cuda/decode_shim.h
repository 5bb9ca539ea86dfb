// What the entry points of decode_cuda.h share.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "shim_device.h"
#include "shim_util.h"
#include "vecops_b200/decode_cuda.h"

namespace vb200 {

struct DecodeDevice {
  int index = -1;
  int sms = 0;
  uint32_t* status = nullptr;
};

// Makes the record's device current (the caller holds a DeviceRestore) and fetches what launches there need.
inline int32_t decode_enter(int32_t device_index, DecodeDevice* device, VecopsError* error) {
  if (vecops_b200_device_count() == 0)
    return set_error(error, VECOPS_STATUS_EXECUTION_ERROR, "no usable CUDA device; there is no CPU fallback");
  if (device_index >= 0) {
    const cudaError_t status = cudaSetDevice(device_index);
    if (status != cudaSuccess) {
      (void)cudaGetLastError();
      return set_error(error, VECOPS_STATUS_EXECUTION_ERROR, "cudaSetDevice(%d): %s", device_index, cudaGetErrorString(status));
    }
    device->index = device_index;
  } else {
    const cudaError_t status = cudaGetDevice(&device->index);
    if (status != cudaSuccess) return set_error(error, VECOPS_STATUS_EXECUTION_ERROR, "cudaGetDevice: %s", cudaGetErrorString(status));
  }
  int major = 0;
  const int32_t rc = shim_device_facts(device->index, &device->sms, &major, &device->status, error);
  if (rc != VECOPS_STATUS_OK) return rc;
  if (major != 10) return set_error(error, VECOPS_STATUS_EXECUTION_ERROR, "the kernels are sm_100a code, device %d is sm_%dx", device->index, major);
  return VECOPS_STATUS_OK;
}

// Counts the launch just made and reports its error; then, unless the call is asynchronous, waits for the stream.
inline int32_t decode_launched(const char* what, VecopsError* error) {
  g_launches.fetch_add(1);
  const cudaError_t status = cudaGetLastError();
  if (status != cudaSuccess) return set_error(error, VECOPS_STATUS_EXECUTION_ERROR, "%s launch: %s", what, cudaGetErrorString(status));
  return VECOPS_STATUS_OK;
}

inline int32_t decode_finish(const char* what, uint32_t flags, void* stream, int device, VecopsError* error) {
  if ((flags & VECOPS_B200_MATMUL_FLAG_ASYNC) != 0) return VECOPS_STATUS_OK;
  const cudaError_t status = cudaStreamSynchronize(static_cast<cudaStream_t>(stream));
  if (status != cudaSuccess) return set_error(error, VECOPS_STATUS_EXECUTION_ERROR, "%s: %s", what, cudaGetErrorString(status));
  if (const uint32_t word = shim_take_status(device))
    return set_error(error, VECOPS_STATUS_EXECUTION_ERROR, "%s on device %d: a bounded device wait ran out (status 0x%x)", what, device, word);
  return VECOPS_STATUS_OK;
}

inline bool decode_aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

}  // namespace vb200
