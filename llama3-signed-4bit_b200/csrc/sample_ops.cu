// Batched sampling behind the C ABI (llama_sample_rows): temperature, top-k, top-p and min-p from
// given random numbers, one id per row of logits.
//
// Logits at or below -1e30 and NaN are masked (the rule of the library's argmax).  With
// w_i = exp((l_i - max) / T) and the ids ordered by logit (descending) and index (ascending), each
// rule keeps a prefix of that order; the kept set is the shortest one.  The draw is the first kept
// id, in index order, whose running mass exceeds uniform x (kept mass).
//
// A draw next to a border of two ids, and the border of a top-p set, must not depend on the order
// of a sum: every weight is rounded once to a multiple of 2^-44 (from a 64-bit exponential) and all
// masses are 64-bit integers (up to 2^18 weights of at most 2^44), whose sums are exact in any order.
//
// One thread-block cluster per row.  Each CTA reads its part of the row once from memory and keeps it
// in shared memory as order-preserving 32-bit keys; everything after that runs on the keys, so the
// bytes of the logits are the only traffic.  A prefix's border (an id) is found by selection, not
// by sorting the row: a histogram over bins of the logit's distance from the maximum (counts for
// top-k; counts and masses for top-p), merged over the cluster through distributed shared memory,
// names the bin that holds the border; bins of more than kList ids are cut further by the bits of
// (key, index); the ids of the last bin are gathered and sorted.  What bounds it: the latency of
// those steps for few rows, the exponentials (64-bit) and the reads for many.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "ops.h"

#define LE_API extern "C" __attribute__((visibility("default")))

namespace le {
namespace sampling {

namespace cg = cooperative_groups;
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

constexpr int kThreads = 512;
constexpr int kBins = 512;    // one per thread
constexpr int kList = 1024;   // ids of a border's bin that are sorted
constexpr int kMaxCluster = 8;

// 2^44 2^y rounded to an integer, for y <= 0: y = n + i / 64 + f with |f| <= 1 / 128, a table of
// 2^(i / 64) and the Taylor series of 2^f to the fifth power (error 4e-17 relative), the method of
// Tang (ACM TOMS 15, 1989).
__device__ __forceinline__ u64 exp2_fixed(double y, const double* table) {
  if (!(y > -46.0)) return 0;
  constexpr double kShift = 6755399441055744.0 / 64.0;  // 1.5 2^52 / 64: adding it rounds y to 1/64
  const double r = y + kShift;
  const int k = (int)(uint32_t)__double_as_longlong(r);  // 64 n + i
  const double f = y - (r - kShift);
  constexpr double c1 = 0.69314718055994530942, c2 = c1 * c1 / 2, c3 = c2 * c1 / 3, c4 = c3 * c1 / 4, c5 = c4 * c1 / 5;
  double p = fma(fma(fma(fma(c5, f, c4), f, c3), f, c2), f, c1);
  const double t = table[k & 63];
  p = fma(t * f, p, t);                                                          // 2^(i / 64 + f)
  const long long e = (long long)((k >> 6) + 44) * (1ll << 52);                       // n + 44, below 2^52
  const double w = __longlong_as_double(__double_as_longlong(p) + e);            // exact: an exponent's change
  return (u64)__double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull;  // + 2^52: nearest integer
}

// What the weights of a row need.
struct Scale {
  uint32_t kmax;
  double mx, c;    // maximum, log2(e) / T
  float inv;       // bins per unit of distance from the maximum
  float fmx;
};
__device__ __forceinline__ u64 weight_of(uint32_t key, const Scale& S, const double* table) {
  if (key == S.kmax) return (u64)kOne;
  if (S.fmx == INFINITY) return 0;  // beside a +inf only its equals have weight
  return exp2_fixed(((double)logit_of(key) - S.mx) * S.c, table);
}
// Bin of a key by its distance from the maximum: falls with the key, 0 for the maximum.
__device__ __forceinline__ int bin_of(uint32_t key, const Scale& S) {
  if (key == S.kmax) return 0;
  return (int)fminf((S.fmx - logit_of(key)) * S.inv, (float)(kBins - 1));
}
// (key, index) as one number: larger = earlier in the order.
__device__ __forceinline__ u64 comp_of(uint32_t key, uint32_t index) { return ((u64)key << 32) | ~index; }

// Inclusive scan of v over the block's 512 threads; *total gets the sum.  red: 16 words.
__device__ __forceinline__ u64 block_scan(u64 v, u64* red, u64* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  __syncthreads();
  if (lane == 31) red[warp] = v;
  __syncthreads();
  u64 before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    const u64 x = red[w];
    if (w < warp) before += x;
    all += x;
  }
  *total = all;
  return v + before;
}

struct Shared {
  uint32_t cnt[2][kBins], lo[2][kBins], hi[2][kBins];  // histograms (masses as two words), used in turn
  u64 list[kList];
  double table[64];
  u64 red[kThreads / 32];
  u64 best[kMaxCluster];                               // of every CTA of the cluster, written by that CTA
  uint32_t low[kMaxCluster], valid[kMaxCluster];
  u64 mass[kMaxCluster];
  u64 rem, answer;
  int bin, n, base, used;
};

// The row's part of one CTA: keys [0, n) are ids first .. first + n - 1; a thread owns `chunk`
// consecutive ones (odd: no bank conflicts), so that scans over the threads are in index order.
struct Part {
  const uint32_t* keys;
  int first, n, begin, end;
};

// The last id (as comp_of) of the shortest prefix, among the ids >= floor_, of `count` ids (by_mass
// false) or of a mass of p x (all their mass).  Called by every thread of the cluster.
__device__ u64 find_border(Shared& sh, const Part& P, const Scale& S, u64 floor_, bool by_mass, u64 count, float p,
                           int& buf) {
  cg::cluster_group cl = cg::this_cluster();
  const int tid = threadIdx.x, ranks = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  u64 target = count, prefix = 0;
  int level = 0, bin0 = 0, shift = 0;
  // digits of (key, index) after the first level; the index's upper bits are all alike
  auto next_shift = [](int l) { return l == 1 ? 55 : l == 2 ? 46 : l == 3 ? 37 : l == 4 ? 32 : 9; };
  auto inside = [&](uint32_t key, u64 c) {
    return key != 0u && c >= floor_ && (level == 0 || (bin_of(key, S) == bin0 && (level == 1 || (c >> shift) == prefix)));
  };
  while (true) {
    buf ^= 1;
    sh.cnt[buf][tid] = 0;
    sh.lo[buf][tid] = 0;
    sh.hi[buf][tid] = 0;
    if (tid == 0) sh.used = 0;
    __syncthreads();
    const int sn = next_shift(level);
    for (int i = P.begin; i < P.end; ++i) {
      const uint32_t key = P.keys[i];
      const u64 c = comp_of(key, (uint32_t)(P.first + i));
      if (!inside(key, c)) continue;
      const int b = level == 0 ? bin_of(key, S) : kBins - 1 - (int)((c >> sn) & (sn == 32 ? 31 : kBins - 1));
      atomicAdd(&sh.cnt[buf][b], 1u);
      if (by_mass) {
        const u64 w = weight_of(key, S, sh.table);
        const uint32_t wl = (uint32_t)w, old = atomicAdd(&sh.lo[buf][b], wl);
        const uint32_t wh = (uint32_t)(w >> 32) + (old + wl < old ? 1u : 0u);
        if (wh) atomicAdd(&sh.hi[buf][b], wh);
      }
    }
    cl.sync();
    u64 n = 0, m = 0, below = 0;
    for (int r = 0; r < ranks; ++r) {
      const Shared* o = cl.map_shared_rank(&sh, r);
      const uint32_t x = o->cnt[buf][tid];
      n += x;
      if (r < rank) below += x;
      if (by_mass) m += ((u64)o->hi[buf][tid] << 32) + o->lo[buf][tid];
    }
    u64 total;
    const u64 v = by_mass ? m : n;
    const u64 cum = block_scan(v, sh.red, &total);
    if (level == 0 && by_mass) {
      const double goal = p > 0.0f ? ceil((double)p * (double)total) : 1.0;
      target = goal < 1.0 ? 1 : (u64)goal;
      if (target > total) target = total;
    }
    if (cum >= target && cum - v < target) {  // one thread
      sh.bin = tid;
      sh.n = (int)n;
      sh.base = (int)below;
      sh.rem = target - (cum - v);
    }
    __syncthreads();
    target = sh.rem;
    if (level == 0) bin0 = sh.bin;
    else {
      const u64 digit = (u64)(kBins - 1 - sh.bin) & (sn == 32 ? 31 : kBins - 1);
      // the digits above sn are those of the prefix; between the key and the index all bits are ones
      prefix = level == 1 ? digit : sn == 9 ? (prefix << 23 | (0x3fffull << 9) | digit) : (prefix << (shift - sn) | digit);
      shift = sn;
    }
    ++level;
    if (sh.n <= kList) break;
  }
  // the border's bin: its ids to every CTA's list, behind those of the CTAs before this one
  const int n = sh.n, base = sh.base;
  for (int i = P.begin; i < P.end; ++i) {
    const uint32_t key = P.keys[i];
    const u64 c = comp_of(key, (uint32_t)(P.first + i));
    if (!inside(key, c)) continue;
    const int at = base + atomicAdd(&sh.used, 1);
    for (int r = 0; r < ranks; ++r) cl.map_shared_rank(&sh, r)->list[at] = c;
  }
  cl.sync();
  int size = 2;
  while (size < n) size <<= 1;
  for (int i = n + tid; i < size; i += kThreads) sh.list[i] = 0;
  for (int k = 2; k <= size; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      __syncthreads();
      for (int i = tid; i < size / 2; i += kThreads) {
        const int a = ((i & ~(j - 1)) << 1) | (i & (j - 1)), b = a | j;
        const u64 x = sh.list[a], y = sh.list[b];
        if (((a & k) == 0) == (x < y)) {  // descending
          sh.list[a] = y;
          sh.list[b] = x;
        }
      }
    }
  __syncthreads();
  if (!by_mass) return sh.list[(int)target - 1];
  const u64 w0 = 2 * tid < n ? weight_of((uint32_t)(sh.list[2 * tid] >> 32), S, sh.table) : 0;
  const u64 w1 = 2 * tid + 1 < n ? weight_of((uint32_t)(sh.list[2 * tid + 1] >> 32), S, sh.table) : 0;
  u64 total;
  const u64 cum = block_scan(w0 + w1, sh.red, &total), before = cum - w0 - w1;
  if (before < target && before + w0 >= target) sh.answer = sh.list[2 * tid];
  if (before + w0 < target && cum >= target) sh.answer = sh.list[2 * tid + 1];
  __syncthreads();
  return sh.answer;
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    k_sample_rows(const T* __restrict__ logits, int64_t ld, int vocab, int seg, const float* __restrict__ temperature,
                  const int32_t* __restrict__ top_k, const float* __restrict__ top_p,
                  const float* __restrict__ min_p, const float* __restrict__ uniform, int32_t* __restrict__ out) {
  extern __shared__ __align__(16) uint32_t s_keys[];
  __shared__ Shared sh;
  cg::cluster_group cl = cg::this_cluster();
  const int ranks = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int row = blockIdx.x / ranks, tid = threadIdx.x, lane = tid & 31;
  cl.barrier_arrive();  // waited for before the first access to another CTA's memory
  const float temp = temperature ? temperature[row] : 1.0f;
  const int k = top_k ? top_k[row] : 0;
  const float p = top_p ? top_p[row] : 1.0f, mp = min_p ? min_p[row] : 0.0f, u = uniform[row];
  if (tid < 64) sh.table[tid] = exp2((double)tid / 64.0);
  Part P;
  P.first = rank * seg;
  P.n = max(0, min(vocab - P.first, seg));
  P.keys = s_keys;
  const int chunk = ((seg + kThreads - 1) / kThreads) | 1;
  P.begin = min(tid * chunk, P.n);
  P.end = min(P.begin + chunk, P.n);
  // keys, and (maximum, lowest index), minimum and count of the unmasked
  u64 best = 0;
  uint32_t low = ~0u, valid = 0;
  const T* l = logits + (int64_t)row * ld + P.first;
#pragma unroll 8
  for (int i = tid; i < P.n; i += kThreads) {
    const uint32_t key = key_of(to_f32(l[i]));
    s_keys[i] = key;
    const u64 c = comp_of(key, (uint32_t)(P.first + i));
    best = c > best ? c : best;
    if (key) {
      low = min(low, key);
      ++valid;
    }
  }
  low = __reduce_min_sync(0xffffffffu, low);
  valid = __reduce_add_sync(0xffffffffu, valid);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 x = __shfl_xor_sync(0xffffffffu, best, o);
    best = x > best ? x : best;
  }
  if (lane == 0) {
    sh.red[tid >> 5] = best;
    sh.lo[0][tid >> 5] = low;
    sh.hi[0][tid >> 5] = valid;
  }
  __syncthreads();
  cl.barrier_wait();
  if (tid < ranks) {
    best = 0;
    low = ~0u;
    valid = 0;
    for (int w = 0; w < kThreads / 32; ++w) {
      best = sh.red[w] > best ? sh.red[w] : best;
      low = min(low, sh.lo[0][w]);
      valid += sh.hi[0][w];
    }
    Shared* o = cl.map_shared_rank(&sh, tid);
    o->best[rank] = best;
    o->low[rank] = low;
    o->valid[rank] = valid;
  }
  cl.sync();
  best = 0;
  low = ~0u;
  valid = 0;
  for (int r = 0; r < ranks; ++r) {
    best = sh.best[r] > best ? sh.best[r] : best;
    low = min(low, sh.low[r]);
    valid += sh.valid[r];
  }
  Scale S;
  S.kmax = (uint32_t)(best >> 32);
  if (S.kmax == 0u || !(temp > 0.01f)) {  // nothing unmasked: id 0; greedy: the maximum's lowest index
    if (rank == 0 && tid == 0) out[row] = S.kmax == 0u ? 0 : (int)~(uint32_t)best;
    return;
  }
  S.fmx = logit_of(S.kmax);
  S.mx = (double)S.fmx;
  S.c = 1.4426950408889634074 / (double)temp;
  // bins over the range of the logits, or what of it has weight (exp(-32) < 2^-44)
  S.inv = (float)(kBins - 1) / fminf(32.0f * temp, S.fmx - logit_of(low));
  u64 floor_ = 0;
  int buf = 0;
  if (k > 0 && (uint32_t)k < valid) floor_ = find_border(sh, P, S, 0, false, (u64)k, 1.0f, buf);
  if (p < 1.0f) floor_ = find_border(sh, P, S, floor_, true, 0, p, buf);
  const u64 wmin = mp > 0.0f ? (u64)ceil((double)(mp < 1.0f ? mp : 1.0f) * kOne) : 1;
  auto kept = [&](int i) -> u64 {
    const uint32_t key = P.keys[i];
    if (key == 0u || comp_of(key, (uint32_t)(P.first + i)) < floor_) return 0;
    const u64 w = weight_of(key, S, sh.table);
    return w >= wmin ? w : 0;
  };
  u64 mine = 0;
  for (int i = P.begin; i < P.end; ++i) mine += kept(i);
  u64 total;
  const u64 cum = block_scan(mine, sh.red, &total);
  if (tid < ranks) cl.map_shared_rank(&sh, tid)->mass[rank] = total;
  cl.sync();
  u64 before = 0, all = 0;
  for (int r = 0; r < ranks; ++r) {
    if (r < rank) before += sh.mass[r];
    all += sh.mass[r];
  }
  const double x = u > 0.0f ? (double)u * (double)all : 0.0;
  const u64 goal = x >= (double)all ? all - 1 : min((u64)x, all - 1);
  if (goal < before || goal >= before + total) return;
  // the draw is in this CTA: the thread whose ids hold it, then the id, by that thread's warp
  const u64 left = goal - before;
  const bool owner = left < cum && left >= cum - mine;
  const unsigned hit = __ballot_sync(0xffffffffu, owner);
  if (hit == 0u) return;
  const int src = __ffs(hit) - 1;
  u64 run = __shfl_sync(0xffffffffu, left - (cum - mine), src);  // mass still to pass
  const int b = __shfl_sync(0xffffffffu, P.begin, src), e = __shfl_sync(0xffffffffu, P.end, src);
  for (int i0 = b; i0 < e; i0 += 32) {
    const u64 w = i0 + lane < e ? kept(i0 + lane) : 0;
    u64 c = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 y = __shfl_up_sync(0xffffffffu, c, o);
      if (lane >= o) c += y;
    }
    const unsigned found = __ballot_sync(0xffffffffu, c > run);
    if (found) {
      if (lane == 0) out[row] = P.first + i0 + __ffs(found) - 1;
      return;
    }
    run -= __shfl_sync(0xffffffffu, c, 31);
  }
}

cudaError_t sample_rows(const void* logits, int type, int64_t ld, int rows, int vocab, const float* temperature,
                        const int32_t* top_k, const float* top_p, const float* min_p, const float* uniform,
                        int32_t* out_ids, int dev, cudaStream_t st) {
  // eight CTAs share a row
  const int ranks = kMaxCluster;
  const int seg = (vocab + ranks - 1) / ranks;
  auto launch = [&](auto x) {
    using T = decltype(x);
    const size_t smem = (size_t)seg * 4;
    if (!allow_smem(k_sample_rows<T>, (kMaxVocab / kMaxCluster) * 4, dev)) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(rows * ranks));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)ranks;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_sample_rows<T>, static_cast<const T*>(logits), ld, vocab, seg, temperature, top_k,
                              top_p, min_p, uniform, out_ids);
  };
  const cudaError_t e = type == LLAMA_F32 ? launch(0.0f) : type == LLAMA_F16 ? launch(__half{}) : launch(__nv_bfloat16{});
  return e == cudaSuccess ? cudaGetLastError() : e;
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
  if (rows < 0 || rows > (1 << 27) || vocab < 1 || ld < vocab) return refuse("rows, vocab or ld out of range");
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
  const cudaError_t e = sample_rows(logits, type, ld, rows, vocab, temperature, top_k, top_p, min_p, uniform, out_ids, dev,
                                    static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? 0 : refuse(cudaGetErrorString(e));
}
