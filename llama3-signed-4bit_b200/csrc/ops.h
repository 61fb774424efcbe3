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

// Text of a call's result, or nullptr for success.  The runtime also keeps a failed call's error as
// its last one, where a later check would take it for its own: it is taken out.
inline const char* error_text(cudaError_t e) {
  if (e == cudaSuccess) return nullptr;
  cudaGetLastError();
  return cudaGetErrorString(e);
}

// Dynamic shared memory above 48 KB, allowed once per kernel and device.
template <typename F>
inline bool allow_smem(F* fn, int bytes, int dev) {
  static std::mutex mu;
  static std::map<std::pair<const void*, int>, bool> done;
  std::lock_guard<std::mutex> lk(mu);
  bool& d = done[{reinterpret_cast<const void*>(fn), dev}];
  if (!d) d = !error_text(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  return d;
}

// Launchers of the paged-cache operators for checked arguments (paged_ops.cu); nullptr, or why they
// failed.  chained: the launches may start while the kernel before them runs out (they wait for
// its results themselves).
namespace paged {
constexpr uint32_t kChunkError = 30;  // error word of a wait of the chunk form that ran out
// The chunk form's bounded waits: where it reports one that ran out (nullptr: the rows' NaN alone tell),
// the bound, and (test only) whether its product issuer first waits on a barrier phase that nothing
// completes.
struct Waits {
  uint32_t* error = nullptr;
  unsigned long long ns = 2000000000ull;
  int expire = 0;
};
const char* append_rows(const llama_paged_kv_t* kv, const void* qkv, int type, int64_t ld, int planes,
                        int64_t plane_stride, int rows, int heads, const int32_t* pos, const int32_t* seq,
                        const float* rope_cos, const float* rope_sin, int n_pos, void* q_out, int q_type, int64_t q_ld,
                        cudaStream_t st, bool chained);
// Workspace that covers every call of at most seqs <= rows sequences and max_kv keys.
size_t attention_bytes_max(int head_dim, int kv_heads, int seqs, int max_kv);
const char* attention_rows(const llama_paged_kv_t* kv, int dev, const void* q, int64_t q_ld, int heads,
                           const int32_t* cu_q, const int32_t* kv_len, int rows, int max_q, int max_kv, float scale,
                           void* out, int out_type, int64_t out_ld, void* workspace, const Waits& waits, cudaStream_t st,
                           bool chained);
}  // namespace paged

// llama_sample_rows for checked arguments (sample_ops.cu); nullptr, or why it failed.
namespace sampling {
// The bound on the wait for a row's copy, and (test only) whether it waits on what nothing completes.
struct Waits {
  unsigned long long ns = 4000000000ull;
  int expire = 0;
};
const char* sample_rows(const void* logits, int type, int64_t ld, int rows, int vocab, const float* temperature,
                        const int32_t* top_k, const float* top_p, const float* min_p, const float* uniform,
                        int32_t* out_ids, const Waits& waits, int dev, cudaStream_t st);
}  // namespace sampling

}  // namespace le
