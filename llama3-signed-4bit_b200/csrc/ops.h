// Internal declarations shared by the engine and the isolated operators (paged_ops.cu,
// sample_ops.cu): error text, device selection, and the launchers that both the C entry points and
// the engine's steps call.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <map>
#include <mutex>
#include <string>
#include <utility>

#include "llama_engine.h"

namespace le {

// Message that llama_engine_last_error(NULL) returns.
void set_global_error(const std::string& s);

// Restores the caller's current CUDA device on scope exit.
struct DeviceGuard {
  int prev = -1;
  explicit DeviceGuard(int dev) {
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    if (prev != dev) cudaSetDevice(dev);
  }
  ~DeviceGuard() {
    int cur = -1;
    if (prev >= 0 && cudaGetDevice(&cur) == cudaSuccess && cur != prev) cudaSetDevice(prev);
  }
};

// Device that owns p, or -1 when p is not device (or managed) memory.
inline int device_of(const void* p) {
  cudaPointerAttributes a{};
  if (cudaPointerGetAttributes(&a, p) != cudaSuccess) {
    cudaGetLastError();
    return -1;
  }
  return a.type == cudaMemoryTypeDevice || a.type == cudaMemoryTypeManaged ? a.device : -1;
}

// Dynamic shared memory above 48 KB, allowed once per kernel and device.
template <typename F>
inline bool allow_smem(F* fn, int bytes, int dev) {
  static std::mutex mu;
  static std::map<std::pair<const void*, int>, bool> done;
  std::lock_guard<std::mutex> lk(mu);
  bool& d = done[{reinterpret_cast<const void*>(fn), dev}];
  if (!d) d = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess;
  return d;
}

}  // namespace le
