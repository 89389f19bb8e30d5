// Launch-status bookkeeping shared by the host launchers.
#pragma once

#include <cuda_runtime.h>

#include <atomic>

#include "../../include/t4a_b200.h"

namespace t4a {
namespace runtime {

// Last CUDA error a launcher of this thread observed (reported by t4a_last_cuda_error).
int& last_error();

// Status of the launches just issued on this thread: T4A_ERR_CUDA when the runtime
// reports a launch error.
inline int check_launch() {
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) {
    last_error() = static_cast<int>(err);
    return T4A_ERR_CUDA;
  }
  return T4A_OK;
}

// Allows a kernel its dynamic shared memory, once a device.
template <typename Kernel>
int allow_shared(Kernel kernel, int bytes, std::atomic<unsigned long long>* done) {
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  const unsigned long long bit = 1ull << (device & 63);
  if (err == cudaSuccess && device < 64 && (done->load(std::memory_order_acquire) & bit)) return T4A_OK;
  if (err == cudaSuccess) err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (err != cudaSuccess) {
    last_error() = static_cast<int>(err);
    cudaGetLastError();
    return T4A_ERR_CUDA;
  }
  done->fetch_or(bit, std::memory_order_release);
  return T4A_OK;
}

// Launches a kernel that may be set up while the stream's previous one ends; it waits for that one
// (griddepcontrol.wait) before it writes memory or reads what that one writes.
template <typename Args>
int launch_early(void (*kernel)(Args), unsigned grid, unsigned block, size_t shared, cudaStream_t stream,
                 const Args& args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(grid);
  config.blockDim = dim3(block);
  config.dynamicSmemBytes = shared;
  config.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attr;
  config.numAttrs = 1;
  const cudaError_t err = cudaLaunchKernelEx(&config, kernel, args);
  if (err != cudaSuccess) {
    last_error() = static_cast<int>(err);
    cudaGetLastError();
    return T4A_ERR_CUDA;
  }
  return T4A_OK;
}

}  // namespace runtime
}  // namespace t4a
