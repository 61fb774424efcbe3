// Batched sampling behind the C ABI (llama_sample_rows): temperature, top-k, top-p and min-p from
// given random numbers, one id per row of logits.
//
// Logits at or below -1e30 and NaN are masked (the rule of the library's argmax).  With
// w_i = exp((l_i - max) / T) and the ids ordered by logit (descending) and index (ascending), each
// rule keeps a prefix of that order; the kept set is the shortest one.  The draw is the first kept
// id, in index order, whose running mass exceeds uniform x (kept mass).
//
// A draw next to a border of two ids, and the border of a top-p set, must not depend on the order
// of a sum: every weight is rounded once to a multiple of 2^-44 (from a 64-bit exp) and all masses
// are 64-bit integers (up to 2^18 weights of at most 2^44), whose sums are exact in any order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "ops.h"

#define LE_API extern "C" __attribute__((visibility("default")))

namespace le {
namespace sampling {

typedef unsigned long long u64;
constexpr int kMaxVocab = 1 << 18;
constexpr double kOne = 17592186044416.0;  // 2^44, the weight of the row's maximum

template <typename T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32(float x) { return x; }
template <> __device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

// Order-preserving key of a logit; 0 = masked.  Adding 0 makes -0 and +0 one value.
__device__ __forceinline__ uint32_t key_of(float l) {
  if (!(l > -1e30f)) return 0u;
  const uint32_t u = __float_as_uint(l + 0.0f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}

// Weight of a key in units of 2^-44, the maximum's being 2^44.
__device__ __forceinline__ u64 weight_of(uint32_t key, float mx, double t) {
  if (key == 0u) return 0;
  const float l = logit_of(key);
  if (l == mx) return (u64)kOne;
  if (mx == INFINITY) return 0;  // beside a +inf only its equals have weight
  const double x = ((double)l - (double)mx) / t;
  return (u64)(exp(x) * kOne + 0.5);
}

__device__ u64 block_sum_u64(u64 v, u64* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  u64 s = 0;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) s += red[w];
  return s;
}

template <typename T>
__global__ void __launch_bounds__(1024)
    k_sample_rows(const T* __restrict__ logits, int64_t ld, int vocab, const float* __restrict__ temperature,
                  const int32_t* __restrict__ top_k, const float* __restrict__ top_p,
                  const float* __restrict__ min_p, const float* __restrict__ uniform, int32_t* __restrict__ out) {
  __shared__ u64 red[32];
  __shared__ u64 s_run;
  __shared__ int s_id;
  const int row = blockIdx.x, tid = threadIdx.x;
  const T* l = logits + (int64_t)row * ld;
  u64 best = 0;  // (key, lowest index) of the maximum
  for (int i = tid; i < vocab; i += blockDim.x) {
    const u64 c = ((u64)key_of(to_f32(l[i])) << 32) | (uint32_t)~i;
    best = c > best ? c : best;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 x = __shfl_xor_sync(0xffffffffu, best, o);
    best = x > best ? x : best;
  }
  if ((tid & 31) == 0) red[tid >> 5] = best;
  __syncthreads();
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) best = red[w] > best ? red[w] : best;
  const uint32_t kmax = (uint32_t)(best >> 32);
  const float temp = temperature ? temperature[row] : 1.0f;
  if (kmax == 0u || !(temp > 0.01f)) {  // nothing unmasked: id 0; greedy: the maximum's lowest index
    if (tid == 0) out[row] = kmax == 0u ? 0 : (int)~(uint32_t)best;
    return;
  }
  const float mx = logit_of(kmax);
  const double t = (double)temp;
  auto mass_from = [&](uint32_t lo) {  // mass of the keys >= lo
    u64 s = 0;
    for (int i = tid; i < vocab; i += blockDim.x) {
      const uint32_t k = key_of(to_f32(l[i]));
      if (k >= lo) s += weight_of(k, mx, t);
    }
    return block_sum_u64(s, red);
  };
  auto count_from = [&](uint32_t lo) {
    u64 s = 0;
    for (int i = tid; i < vocab; i += blockDim.x) s += key_of(to_f32(l[i])) >= lo ? 1 : 0;
    return block_sum_u64(s, red);
  };
  // kept: keys > kt, and the first `ties` ids whose key is kt
  uint32_t kt = 1u;
  u64 ties = ~0ull;
  const int k = top_k ? top_k[row] : 0;
  if (k > 0 && (u64)k < count_from(1u)) {
    kt = 0u;
    for (int b = 31; b >= 0; --b)
      if (count_from(kt | (1u << b)) >= (u64)k) kt |= 1u << b;
    ties = (u64)k - (kt == ~0u ? 0 : count_from(kt + 1u));
  }
  const float p = top_p ? top_p[row] : 1.0f;
  if (p < 1.0f) {
    const u64 at_kt = count_from(kt) - count_from(kt + 1u);
    const u64 spare = (at_kt - (ties < at_kt ? ties : at_kt)) * weight_of(kt, mx, t);  // ties at kt that top-k drops
    const u64 total = mass_from(kt) - spare;
    const double goal = p > 0.0f ? (double)p * (double)total : 0.0;
    u64 need = (u64)ceil(goal);
    need = need < 1 ? 1 : need > total ? total : need;
    uint32_t kp = 0u;
    for (int b = 31; b >= 0; --b) {
      const uint32_t c = kp | (1u << b);
      const u64 m = c > kt ? mass_from(c) : total;
      if (m >= need) kp = c;
    }
    kp = kp < kt ? kt : kp;
    const u64 above = kp == ~0u ? 0 : mass_from(kp + 1u), w = weight_of(kp, mx, t);
    const u64 r = (need - above + w - 1) / w;
    if (kp > kt || r < ties) ties = r;
    kt = kp;
  }
  const float mp = min_p ? min_p[row] : 0.0f;
  const u64 wmin = mp > 0.0f ? (u64)ceil((double)(mp < 1.0f ? mp : 1.0f) * kOne) : 0;
  // two passes in index order over tiles of blockDim ids: the kept mass, then the draw
  u64 total = 0, goal = 0;
  for (int pass = 0; pass < 2; ++pass) {
    u64 run = 0, seen = 0;  // mass and ties before the tile
    for (int i0 = 0; i0 < vocab; i0 += blockDim.x) {
      const int i = i0 + tid;
      const uint32_t key = i < vocab ? key_of(to_f32(l[i])) : 0u;
      u64 w = key >= kt && key > 0u ? weight_of(key, mx, t) : 0;
      if (w < wmin) w = 0;
      // inclusive scan of the ties, then of the kept weights
      const int lane = tid & 31, warp = tid >> 5;
      auto scan = [&](u64 v, u64* sum) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const u64 x = __shfl_up_sync(0xffffffffu, v, o);
          if (lane >= o) v += x;
        }
        __syncthreads();
        if (lane == 31) red[warp] = v;
        __syncthreads();
        u64 all = 0;
        for (int x = 0; x < (int)(blockDim.x >> 5); ++x) {
          if (x < warp) v += red[x];
          all += red[x];
        }
        *sum = all;
        return v;
      };
      u64 tile_ties, tile_mass;
      const u64 rank = seen + scan(key == kt ? 1 : 0, &tile_ties);  // 1-based among the ties
      if (key == kt && rank > ties) w = 0;
      const u64 cum = run + scan(w, &tile_mass);
      if (pass == 1 && w > 0 && cum > goal && cum - w <= goal) out[row] = i;
      seen += tile_ties;
      run += tile_mass;
    }
    if (pass == 0) {
      total = run;
      const float u = uniform[row];
      const double x = u > 0.0f ? (double)u * (double)total : 0.0;
      goal = x >= (double)total ? total - 1 : (u64)x;
      if (goal >= total) goal = total - 1;
    }
  }
}

static int refuse(const char* why, int rc = -1) {
  set_global_error(std::string("llama_sample_rows: ") + why);
  return rc;
}

}  // namespace sampling
}  // namespace le

using namespace le;

LE_API int llama_sample_rows(const void* logits, int type, int64_t ld, int rows, int vocab, const float* temperature,
                             const int32_t* top_k, const float* top_p, const float* min_p, const float* uniform,
                             int32_t* out_ids, void* stream) {
  using namespace sampling;
  if (!logits || !uniform || !out_ids) return refuse("NULL argument");
  if (type != LLAMA_F32 && type != LLAMA_F16 && type != LLAMA_BF16) return refuse("unknown type");
  if (rows < 0 || vocab < 1 || ld < vocab) return refuse("rows, vocab or ld out of range");
  if (vocab > kMaxVocab) return refuse("vocab exceeds the maximum", -2);
  const int size = type == LLAMA_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % size != 0) return refuse("logits are misaligned");
  if (rows == 0) return 0;
  const int dev = device_of(logits);
  const void* ptrs[] = {temperature, top_k, top_p, min_p, uniform, out_ids};
  if (dev < 0) return refuse("every pointer must be memory of one CUDA device");
  for (const void* p : ptrs)
    if (p && device_of(p) != dev) return refuse("every pointer must be memory of one CUDA device");
  DeviceGuard dg(dev);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto launch = [&](auto x) {
    using T = decltype(x);
    k_sample_rows<T><<<rows, 1024, 0, st>>>(static_cast<const T*>(logits), ld, vocab, temperature, top_k, top_p, min_p,
                                            uniform, out_ids);
  };
  if (type == LLAMA_F32) launch(0.0f);
  else if (type == LLAMA_F16) launch(__half{});
  else launch(__nv_bfloat16{});
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : refuse(cudaGetErrorString(e));
}
