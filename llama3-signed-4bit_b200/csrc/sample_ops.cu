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
// One thread-block cluster per row.  Each CTA brings its part of the row into shared memory once (bulk
// copy); everything after that runs there, so the bytes of the logits are the only traffic.
//   * A row without truncation takes one pass of weights, summed per 512 bytes of the row.
//   * A border (top-k, top-p) usually lies among the first ids: a bound on the logit that a few of them
//     reach is taken from a histogram of the threads' maxima, the ids above it are gathered in one
//     CTA, and the rules and the draw run on that list.
//   * Where the list does not reach the border (a wide top-p set, a large top-k, many equal logits), a
//     histogram of the whole row is merged over the cluster through distributed shared memory and names
//     the bin that holds the border; bins of more than kList ids are cut further by the bits of
//     (key, index); the ids of the last bin are gathered.
// No list is sorted: the border, or the draw, in a list is again found by a histogram (of counts or
// masses, over bins in the list's order) and by comparing the few entries of one bin with each other.
// What bounds it: the latency of those steps for few rows.  For many, that a row has an SM to itself, so that
// its copy, its passes and their barriers follow one another (greedy rows, without a weight to compute, take
// twice the copy's time), in two uneven waves of rows; then the weights (nine 64-bit operations and a look-up
// in a table whose entries share banks) and, where the border lies far down, three atomics for each id.
// Device time in us, all rows with the same rule:
//                            greedy  T only  top_k 50  1000  top_p 0.9  0.95, T 1.2
//   1 x 128256 fp32             3.8     9.8      13.5  17.7       17.1           38
//   64 x 128256 fp32            9.6    26.1      29.4  37.3       43.8          105   (32.8 MB: 5.0 at the copy rate)
//   256 x 50257 bf16           10.4    35.5      32.1  86.2       56.7          141   (25.7 MB: 3.9)
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "ops.h"
#include "ptx.cuh"

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
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float x) { return __float2bfloat16_rn(x); }

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 512;
constexpr int kList = 2 * kThreads;  // entries of a list
constexpr int kBorder = 1024;        // ids of a border's bin that are not cut further
constexpr int kTopWanted = 512;  // ids the list is made for when only a mass bounds it
constexpr int kMaxCluster = 8;
constexpr float kMasked = -1e30f;
constexpr u64 kLate = ~0ull;  // in the place of a (key, index)

// Order-preserving key of an unmasked logit.  Adding 0 makes -0 and +0 one value.
__device__ __forceinline__ uint32_t key_of(float l) {
  const uint32_t u = __float_as_uint(l + 0.0f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}
// (key, index) as one number: larger = earlier in the order.
__device__ __forceinline__ u64 comp_of(float l, uint32_t index) { return ((u64)key_of(l) << 32) | ~index; }

constexpr int kTable = 256;

// What the weights and bins of a row need.
struct Scale {
  float top;       // maximum
  float least;     // logits at or below it weigh less than 2^-45
  bool wide;       // least lies below kMasked: masked logits need a check of their own
  double c;        // log2(e) / T
  float inv;       // bins per unit of distance from the maximum
};
// exp((l - top) / T) in units of 2^-44, rounded to an integer: with y = (l - top) c = n + i / 256 + f,
// |f| <= 1 / 512, it is 2^(n + 44) table[i] 2^f, and 2^f is its Taylor series to the fourth power (error
// 4e-17), the method of Tang (ACM TOMS 15, 1989).  The product is rounded by adding it to 2^52.
__device__ __forceinline__ u64 weight_of(float l, const Scale& S, const double* table) {
  if (S.top == INFINITY) return l == S.top ? (u64)kOne : 0;  // beside a +inf only its equals have weight
  constexpr double kShift = 6755399441055744.0 / kTable;     // 1.5 2^52 / 256: adding it rounds to 1/256
  const double d = (double)fmaxf(l, S.least) - (double)S.top;  // NaN counts as least
  const double r = fma(d, S.c, kShift);
  const double f = fma(d, S.c, kShift - r);
  const int k = (int)(uint32_t)__double_as_longlong(r);        // 256 n + i
  constexpr double c1 = 0.69314718055994530942, c2 = c1 * c1 / 2, c3 = c2 * c1 / 3, c4 = c3 * c1 / 4;
  const double q = fma(fma(fma(fma(c4, f, c3), f, c2), f, c1), f, 1.0);
  const double t = table[k & (kTable - 1)];
  const int hi = __double2hiint(t) + ((k >> 8) + 44) * (1 << 20);  // n + 44 on the exponent
  const double w = fma(__hiloint2double(hi, __double2loint(t)), q, 4503599627370496.0);
  const u64 v = (u64)__double_as_longlong(w) & 0xfffffffffffffull;
  return S.wide && !(l > kMasked) ? 0 : v;
}
// Bin of an unmasked logit by its distance from the maximum (0 for the maximum).
__device__ __forceinline__ float place_of(float l, const Scale& S) { return l == S.top ? 0.0f : (S.top - l) * S.inv; }
__device__ __forceinline__ int bin_of(float l, const Scale& S) { return (int)fminf(place_of(l, S), (float)(kBins - 1)); }

struct Shared {
  union {
    struct {
      uint32_t cnt[2][kBins], lo[2][kBins], hi[2][kBins];  // histograms (masses as two words), used in turn
      u64 sum[kBins];                                      // the one that is searched: counts or masses
    };
    u64 vals[kList];                                       // values of the list's entries, after the search
  };
  u64 list[kList];
  double table[kTable];
  u64 red[kWarps];
  uint32_t red32[kWarps];
  u64 best[kMaxCluster], mass[kMaxCluster];            // of every CTA, written by that CTA
  float low[kMaxCluster];
  uint32_t found[kMaxCluster];
  u64 total, rem, answer;
  int bin, used, redo;
};

constexpr int kSharedBytes = (sizeof(Shared) + 15) / 16 * 16;

// Adds w to the two-word sum of a bin.
__device__ __forceinline__ void add_mass(Shared& sh, int buf, int b, u64 w) {
  const uint32_t wl = (uint32_t)w, old = atomicAdd(&sh.lo[buf][b], wl);
  const uint32_t wh = (uint32_t)(w >> 32) + (old + wl < old ? 1u : 0u);
  if (wh) atomicAdd(&sh.hi[buf][b], wh);
}

// The bin of sh.sum in which the running sum reaches a target that goal(total) gives (between 1 and the
// total): sh.bin, what the target has left there (sh.rem) and the total.  One warp, 16 bins a lane.
template <typename F>
__device__ __forceinline__ void search_bins(Shared& sh, F goal) {
  __syncthreads();
  if (threadIdx.x < 32) {
    constexpr int kPer = kBins / 32;
    const int lane = threadIdx.x;
    u64 mine = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) mine += sh.sum[lane * kPer + i];
    u64 cum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 y = __shfl_up_sync(0xffffffffu, cum, o);
      if (lane >= o) cum += y;
    }
    const u64 total = __shfl_sync(0xffffffffu, cum, 31), target = goal(total);
    u64 left = target - (cum - mine);
    if (cum >= target && cum - mine < target) {
      int i = 0;
      while (i < kPer - 1 && left > sh.sum[lane * kPer + i]) left -= sh.sum[lane * kPer + i++];
      sh.bin = lane * kPer + i;
      sh.rem = left;
    }
    if (lane == 0) {
      sh.total = total;
      sh.used = 0;
    }
  }
  __syncthreads();
}

// A list entry of a thread: place in the order (larger is earlier; 0: none), value, and its bin.
struct Entry {
  u64 order, value;
  int bin;
};
// The order of the entry at which the running sum of the values reaches goal(total).  Two entries a
// thread; bins rise as the order falls.
template <typename F>
__device__ u64 select(Shared& sh, const Entry (&e)[2], int& buf, F goal) {
  buf ^= 1;
  const int tid = threadIdx.x;
  if (tid < kBins) sh.lo[buf][tid] = sh.hi[buf][tid] = 0;
  __syncthreads();
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (e[h].order) add_mass(sh, buf, e[h].bin, e[h].value);
  __syncthreads();
  if (tid < kBins) sh.sum[tid] = ((u64)sh.hi[buf][tid] << 32) + sh.lo[buf][tid];
  search_bins(sh, goal);
  const int bin = sh.bin;
  int at[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    at[h] = e[h].order && e[h].bin == bin ? atomicAdd(&sh.used, 1) : -1;
    if (at[h] >= 0) {
      sh.list[at[h]] = e[h].order;
      sh.vals[at[h]] = e[h].value;
    }
  }
  __syncthreads();
  const int n = sh.used;
  const u64 rem = sh.rem;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (at[h] < 0) continue;
    u64 before = 0;
    for (int i = 0; i < n; ++i) before += sh.list[i] > e[h].order ? sh.vals[i] : 0;
    if (before < rem && before + e[h].value >= rem) sh.answer = e[h].order;
  }
  __syncthreads();
  return sh.answer;
}

// Sum over the block's threads.
__device__ __forceinline__ u64 block_sum(u64 v, u64* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A CTA's part of the row in shared memory: 16-byte runs, a warp's 32 neighbouring ones a group of 512
// bytes, `groups` consecutive groups for every warp, so that sums over (warp, group) are in index order.
// Slots before and behind the part hold -inf.
template <typename T>
struct Part {
  static constexpr int kRun = 16 / (int)sizeof(T);
  const uint8_t* base;
  int groups, id0;  // id0: id of slot 0
  __device__ __forceinline__ void run(int group, int lane, float (&x)[kRun]) const {
    const uint4 u = *reinterpret_cast<const uint4*>(base + group * 512 + lane * 16);
    if constexpr (sizeof(T) == 4) {
      x[0] = __uint_as_float(u.x); x[1] = __uint_as_float(u.y); x[2] = __uint_as_float(u.z); x[3] = __uint_as_float(u.w);
    } else {
      const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int i = 0; i < kRun; ++i) x[i] = to_f32(e[i]);
    }
  }
  __device__ __forceinline__ uint32_t id(int group, int lane, int e) const { return id0 + (group * 32 + lane) * kRun + e; }
  // Sum of the thread's weights; no branch, so that the exponentials of a run overlap.
  __device__ __forceinline__ u64 mass(const Scale& S, const double* table, int g) const {
    float x[kRun];
    run((threadIdx.x >> 5) * groups + g, threadIdx.x & 31, x);
    u64 w = 0;
#pragma unroll
    for (int e = 0; e < kRun; ++e) w += weight_of(x[e], S, table);
    return w;
  }
  // f(logit, id) for every unmasked element of the thread
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int g = 0; g < groups; ++g) {
      float x[kRun];
      run(warp * groups + g, lane, x);
#pragma unroll
      for (int e = 0; e < kRun; ++e)
        if (x[e] > kMasked) f(x[e], id(warp * groups + g, lane, e));
    }
  }
};

__device__ __forceinline__ float logit_of_comp(u64 c) { return logit_of((uint32_t)(c >> 32)); }
// Mass that a top-p set has to reach.
__device__ __forceinline__ u64 need_of(float p, u64 total) {
  const double goal = p > 0.0f ? ceil((double)p * (double)total) : 1.0;
  const u64 n = goal < 1.0 ? 1 : (u64)goal;
  return n > total ? total : n;
}
// The point of a kept mass that a random number falls on.
__device__ __forceinline__ u64 goal_of(float u, u64 total) {
  const double x = u > 0.0f ? (double)u * (double)total : 0.0;
  return x >= (double)total ? total - 1 : min((u64)x, total - 1);
}

// The last id (as comp_of) of the shortest prefix, among the ids >= floor_, of `count` ids (by_mass
// false) or of a mass of p x (all their mass).  Called by every thread of the cluster.
template <int R, typename T>
__device__ u64 find_border(Shared& sh, const Part<T>& P, const Scale& S, u64 floor_, bool by_mass, u64 count, float p,
                           int& buf) {
  cg::cluster_group cl = cg::this_cluster();
  const int tid = threadIdx.x, rank = (int)cl.block_rank();
  u64 target = count, prefix = 0;
  int level = 0, bin0 = 0, shift = 0;
  // digits of (key, index) after the first level; the index's upper bits are all alike
  auto next_shift = [](int l) { return l == 1 ? 55 : l == 2 ? 46 : l == 3 ? 37 : l == 4 ? 32 : 9; };
  auto inside = [&](float l, u64 c) {
    return c >= floor_ && (level == 0 || (bin_of(l, S) == bin0 && (level == 1 || (c >> shift) == prefix)));
  };
  while (true) {
    buf ^= 1;
    if (tid < kBins) {
      sh.cnt[buf][tid] = 0;
      sh.lo[buf][tid] = 0;
      sh.hi[buf][tid] = 0;
    }
    if (tid == 0) sh.used = 0;
    __syncthreads();
    const int sn = next_shift(level);
    for (int g = 0; g < P.groups; ++g) {
      float x[Part<T>::kRun];
      const int group = (tid >> 5) * P.groups + g;
      P.run(group, tid & 31, x);
      bool in[Part<T>::kRun];
      bool some = false;
#pragma unroll
      for (int e = 0; e < Part<T>::kRun; ++e) {
        in[e] = x[e] > kMasked && inside(x[e], comp_of(x[e], P.id(group, tid & 31, e)));
        some |= in[e];
      }
      if (!some) continue;
      u64 w[Part<T>::kRun];
      if (by_mass) {  // no branch between them: the exponentials of a run overlap
#pragma unroll
        for (int e = 0; e < Part<T>::kRun; ++e) w[e] = weight_of(x[e], S, sh.table);
      }
#pragma unroll
      for (int e = 0; e < Part<T>::kRun; ++e) {
        if (!in[e]) continue;
        const u64 c = comp_of(x[e], P.id(group, tid & 31, e));
        const int b = level == 0 ? bin_of(x[e], S) : kBins - 1 - (int)((c >> sn) & (sn == 32 ? 31 : kBins - 1));
        atomicAdd(&sh.cnt[buf][b], 1u);
        if (by_mass) {
          const uint32_t wl = (uint32_t)w[e], old = atomicAdd(&sh.lo[buf][b], wl);
          const uint32_t wh = (uint32_t)(w[e] >> 32) + (old + wl < old ? 1u : 0u);
          if (wh) atomicAdd(&sh.hi[buf][b], wh);
        }
      }
    }
    cl.sync();
    uint32_t below = 0, n = 0;
    if (tid < kBins) {
      u64 m = 0;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const Shared* o = cl.map_shared_rank(&sh, r);
        const uint32_t x = o->cnt[buf][tid];
        n += x;
        if (r < rank) below += x;
        if (by_mass) m += ((u64)o->hi[buf][tid] << 32) + o->lo[buf][tid];
      }
      sh.sum[tid] = by_mass ? m : n;
    }
    search_bins(sh, [&](u64 total) { return level > 0 ? target : by_mass ? need_of(p, total) : min(target, total); });
    target = sh.rem;
    if (tid == sh.bin) {
      sh.red32[0] = n;
      sh.red32[1] = below;
    }
    if (level == 0) {
      bin0 = sh.bin;
    } else {
      const u64 digit = (u64)(kBins - 1 - sh.bin) & (sn == 32 ? 31 : kBins - 1);
      // the digits above sn are those of the prefix; between the key and the index all bits are ones
      prefix = level == 1 ? digit : sn == 9 ? (prefix << 23 | (0x3fffull << 9) | digit) : (prefix << (shift - sn) | digit);
      shift = sn;
    }
    ++level;
    __syncthreads();
    if (sh.red32[0] <= kBorder) break;
  }
  // the border's bin: its ids to every CTA's list, behind those of the CTAs before this one
  const int n = (int)sh.red32[0], base = (int)sh.red32[1];
  P.each([&](float l, uint32_t id) {
    const u64 c = comp_of(l, id);
    if (!inside(l, c)) return;
    const int at = base + atomicAdd(&sh.used, 1);
#pragma unroll
    for (int r = 0; r < R; ++r) cl.map_shared_rank(&sh, r)->list[at] = c;
  });
  cl.sync();
  Entry e[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    e[h].order = 2 * tid + h < n ? sh.list[2 * tid + h] : 0;
    const float l = logit_of_comp(e[h].order);
    e[h].value = !e[h].order ? 0 : by_mass ? weight_of(l, S, sh.table) : 1;
    // the bin's own bins
    e[h].bin = (int)fminf(fmaxf((place_of(l, S) - (float)bin0) * (float)kBins, 0.0f), (float)(kBins - 1));
  }
  return select(sh, e, buf, [&](u64) { return target; });
}

// The rules and the draw on a list of the row's first n ids (c: two a thread, 0: none): writes the id, or
// returns false when the list ends before the top-p border.  all: mass of the row (top-k off).
__device__ bool draw_from_list(Shared& sh, const Scale& S, const u64 (&c)[2], int n, int k, float p, u64 all, u64 wmin,
                               float u, int32_t* out) {
  int buf = 0;
  Entry e[2];
  u64 w[2], floor_ = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float l = logit_of_comp(c[h]);
    w[h] = c[h] ? weight_of(l, S, sh.table) : 0;
    e[h] = {c[h], 1, c[h] ? bin_of(l, S) : 0};
  }
  if (k > 0 && k < n) floor_ = select(sh, e, buf, [&](u64) { return (u64)k; });
  if (p < 1.0f) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      e[h].order = c[h] >= floor_ && w[h] > 0 ? c[h] : 0;
      e[h].value = w[h];
    }
    const u64 need = k > 0 ? 0 : need_of(p, all);
    floor_ = select(sh, e, buf, [&](u64 total) { return k > 0 ? need_of(p, total) : need > total ? total : need; });
    if (need > sh.total) return false;  // uniform
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    e[h].order = c[h] >= floor_ && c[h] && w[h] >= wmin ? (uint32_t)c[h] : 0;  // ~index
    e[h].value = w[h];
    e[h].bin = (int)(~(uint32_t)c[h] >> 9) & (kBins - 1);
  }
  const u64 id = select(sh, e, buf, [&](u64 total) { return goal_of(u, total) + 1; });
  if (threadIdx.x == 0) *out = (int32_t)~(uint32_t)id;
  return true;
}

template <int R, typename T>
__global__ void __launch_bounds__(kThreads)
    k_sample_rows(const T* __restrict__ logits, int64_t ld, int vocab, int seg, int groups,
                  const float* __restrict__ temperature, const int32_t* __restrict__ top_k,
                  const float* __restrict__ top_p, const float* __restrict__ min_p, const float* __restrict__ uniform,
                  int32_t* __restrict__ out, Waits W) {
  extern __shared__ __align__(16) uint8_t s_dyn[];
  Shared& sh = *reinterpret_cast<Shared*>(s_dyn);
  uint8_t* const s_part = s_dyn + kSharedBytes;
  __shared__ __align__(8) u64 s_bar, s_never;  // the copy's, and (test only) one that nothing completes
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), row = blockIdx.x / R, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  cl.barrier_arrive();  // waited for before the first access to another CTA's memory
  // the part [first, first + n) of the row, at the 16-byte phase it has in memory: its aligned middle by
  // one bulk copy, the ends element by element
  const int first = rank * seg, n = max(0, min(vocab - first, seg));
  const T* src = logits + (int64_t)row * ld + first;
  const int off = (int)((reinterpret_cast<uintptr_t>(src) & 15u) / sizeof(T));
  constexpr int kRun = Part<T>::kRun;
  const int head = off ? min(n, kRun - off) : 0, body = (n - head) / kRun * kRun;
  T* slots = reinterpret_cast<T*>(s_part);
  if (tid == 0) {
    mbar_init(smem_u32(&s_bar), 1);
    mbar_init(smem_u32(&s_never), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    mbar_expect_tx(smem_u32(&s_bar), (uint32_t)body * sizeof(T));
    if (body) bulk_g2s(smem_u32(slots + off + head), src + head, (uint32_t)body * sizeof(T), smem_u32(&s_bar));
  }
  if (tid < head) slots[off + tid] = src[tid];
  if (tid < n - head - body) slots[off + head + body + tid] = src[head + body + tid];
  if (tid < off) slots[tid] = from_f32<T>(-INFINITY);
  for (int i = off + n + tid; i < groups * kWarps * 32 * kRun; i += kThreads) slots[i] = from_f32<T>(-INFINITY);
  Part<T> P;
  P.base = s_part;
  P.groups = groups;
  P.id0 = first - off;
  const float temp = temperature ? temperature[row] : 1.0f;
  const int k = top_k ? top_k[row] : 0;
  const float p = top_p ? top_p[row] : 1.0f, mp = min_p ? min_p[row] : 0.0f, u = uniform[row];
  if (tid < kTable) sh.table[tid] = exp2((double)tid / kTable);
  __syncthreads();
  auto wait = [&](u64* bar) {
    const unsigned long long t0 = gtimer();
    while (!mbar_try(smem_u32(bar), 0))
      if (gtimer() - t0 > W.ns) return false;
    return true;
  };
  bool late = !wait(W.expire ? &s_never : &s_bar);  // no copy within the bound: the row's id becomes -1
  if (late) wait(&s_bar);  // once more: it shall not land where another CTA's memory is by then
  // maximum with its lowest index (of the unmasked), and the lowest of the threads' maxima
  float mine = kMasked;
  uint32_t at = 0;
  for (int g = 0; g < groups; ++g) {
    float x[kRun];
    P.run(warp * groups + g, lane, x);
    const uint32_t id = P.id(warp * groups + g, lane, 0);
#pragma unroll
    for (int e = 0; e < kRun; ++e)
      if (x[e] > mine) {
        mine = x[e];
        at = id + e;
      }
  }
  const bool any = mine > kMasked;
  u64 best = any ? comp_of(mine, at) : 0;
  float low = any ? mine : INFINITY;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 x = __shfl_xor_sync(0xffffffffu, best, o);
    best = x > best ? x : best;
    low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
  }
  late = __any_sync(0xffffffffu, late);
  if (lane == 0) {
    sh.red[warp] = late ? kLate : best;
    sh.red32[warp] = __float_as_uint(low);
  }
  if (tid < kBins) sh.cnt[1][tid] = 0;
  if (tid == 0) sh.used = 0;
  __syncthreads();
  cl.barrier_wait();
  if (warp == 0) {
    best = sh.red[lane];
    low = __uint_as_float(sh.red32[lane]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const u64 x = __shfl_xor_sync(0xffffffffu, best, o);
      best = x > best ? x : best;
      low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
    }
    if (lane < R) {
      Shared* o = cl.map_shared_rank(&sh, lane);
      o->best[rank] = best;
      o->low[rank] = low;
    }
  }
  cl.sync();
  best = 0;
  low = INFINITY;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    best = sh.best[r] > best ? sh.best[r] : best;
    low = fminf(low, sh.low[r]);
  }
  if (best == kLate || best == 0 || !(temp > 0.01f)) {
    // the copy did not come; nothing unmasked: id 0; greedy: the maximum's lowest index
    if (rank == 0 && tid == 0) out[row] = best == kLate ? -1 : best == 0 ? 0 : (int)~(uint32_t)best;
    return;
  }
  Scale S;
  S.top = logit_of((uint32_t)(best >> 32));
  S.c = 1.4426950408889634074 / (double)temp;
  // rounded down, and below top whatever fp32's (or fp64's) spacing there.  Where a spacing is so many
  // temperatures that least would leave the exponent's range, nothing lies between it and top: any
  // smaller distance that rounds to no weight will do.
  S.least = fminf(__double2float_rd(fmax((double)S.top - 50.0 / S.c, -3.0e38)), nextafterf(S.top, -INFINITY));
  const double reach = (double)S.top - (double)S.least;
  if (reach * S.c > 900.0) S.c = 900.0 / reach;
  S.wide = !(S.least > kMasked);
  // bins over somewhat more than the range of the threads' maxima, or over what has weight
  // (exp(-32) < 2^-44); what lies below shares the last bin
  S.inv = (float)(kBins - 1) / fminf(32.0f * temp, 1.6f * (S.top - low));
  const u64 wmin = mp > 0.0f ? (u64)ceil((double)(mp < 1.0f ? mp : 1.0f) * kOne) : 1;
  const bool by_k = k > 0 && k < vocab;
  u64 floor_ = 0;
  int buf = 0;
  if (by_k || p < 1.0f) {
    // ---- the list: ids down to the bin that holds the wanted number of threads' maxima ----
    if (any) atomicAdd(&sh.cnt[1][bin_of(mine, S)], 1u);
    if (!by_k) {
      u64 part = 0;
      for (int g = 0; g < groups; ++g) part += P.mass(S, sh.table, g);
      part = block_sum(part, sh.red);
      if (tid < R) cl.map_shared_rank(&sh, tid)->mass[rank] = part;
    }
    cl.sync();
    if (tid < kBins) {
      uint32_t v = 0;
#pragma unroll
      for (int r = 0; r < R; ++r) v += cl.map_shared_rank(&sh, r)->cnt[1][tid];
      sh.sum[tid] = v;
    }
    const u64 wanted = by_k ? (u64)k : (u64)kTopWanted;
    search_bins(sh, [&](u64 total) { return min(total, wanted); });
    const int bin = by_k && sh.total < wanted ? kBins - 1 : sh.bin;
    // straight into the first CTA's list, every CTA in a region of its own
    constexpr int kRegion = kList / R;
    if (any && bin_of(mine, S) <= bin) {
      u64* to = cl.map_shared_rank(&sh, 0)->list + rank * kRegion;
      P.each([&](float l, uint32_t id) {
        if (bin_of(l, S) > bin) return;
        const int i = atomicAdd(&sh.used, 1);
        if (i < kRegion) to[i] = comp_of(l, id);
      });
    }
    __syncthreads();
    if (tid < R) cl.map_shared_rank(&sh, tid)->found[rank] = (uint32_t)sh.used;
    cl.sync();
    uint32_t ids = 0;
    bool fits = true;
    u64 all = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      ids += sh.found[r];
      fits &= sh.found[r] <= kRegion;
      if (!by_k) all += sh.mass[r];
    }
    if (fits) {  // the same in every CTA
      if (rank == 0) {
        u64 c[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int i = tid + h * kThreads;
          c[h] = i % kRegion < (int)sh.found[i / kRegion] ? sh.list[i] : 0;
        }
        const bool done = draw_from_list(sh, S, c, (int)ids, by_k ? k : 0, p, all, wmin, u, out + row);
        if (tid < R) cl.map_shared_rank(&sh, tid)->redo = done ? 0 : 1;
      }
      cl.sync();
      if (!sh.redo) return;
    }
    if (by_k) floor_ = find_border<R>(sh, P, S, 0, false, (u64)k, 1.0f, buf);
    if (p < 1.0f) floor_ = find_border<R>(sh, P, S, floor_, true, 0, p, buf);
    __syncthreads();
  }
  // ---- the kept mass of every group, then the group, the run and the id of the draw ----
  auto kept = [&](float l, uint32_t id) -> u64 {
    if (!(l > kMasked) || comp_of(l, id) < floor_) return 0;
    const u64 w = weight_of(l, S, sh.table);
    return w >= wmin ? w : 0;
  };
  for (int g = 0; g < groups; ++g) {
    u64 w = 0;
    if (floor_ == 0 && wmin == 1) {
      w = P.mass(S, sh.table, g);
    } else {
      float x[kRun];
      P.run(warp * groups + g, lane, x);
#pragma unroll
      for (int e = 0; e < kRun; ++e) w += kept(x[e], P.id(warp * groups + g, lane, e));
    }
    // at most 8 x 2^44 a lane: two words of 24 bits
    const u64 a = __reduce_add_sync(0xffffffffu, (uint32_t)w & 0xffffffu), b = __reduce_add_sync(0xffffffffu, (uint32_t)(w >> 24));
    if (lane == 0) sh.list[warp * groups + g] = (b << 24) + a;
  }
  __syncthreads();
  if (tid < kBins) sh.sum[tid] = tid < kWarps * groups ? sh.list[tid] : 0;
  __syncthreads();
  if (warp > 0) {
    cl.sync();
    return;
  }
  // one warp: the CTA's mass, the point of the row's, and the group that holds it
  u64 part = 0;
#pragma unroll
  for (int i = 0; i < kBins / 32; ++i) part += sh.sum[lane * (kBins / 32) + i];
  u64 cum = part;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 y = __shfl_up_sync(0xffffffffu, cum, o);
    if (lane >= o) cum += y;
  }
  const u64 total = __shfl_sync(0xffffffffu, cum, 31);
  if (lane < R) cl.map_shared_rank(&sh, lane)->mass[rank] = total;
  cl.sync();
  u64 before = 0, all = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (r < rank) before += sh.mass[r];
    all += sh.mass[r];
  }
  u64 left = goal_of(u, all) - before;  // wraps where the draw is in an earlier CTA
  const unsigned hit = __ballot_sync(0xffffffffu, left < cum && left >= cum - part && left < total);
  if (hit == 0u) return;
  const int owner = __ffs(hit) - 1;
  left -= __shfl_sync(0xffffffffu, cum - part, owner);
  int group = owner * (kBins / 32);
  while (left >= sh.sum[group]) left -= sh.sum[group++];
  float x[kRun];
  P.run(group, lane, x);
  u64 sum = 0;
#pragma unroll
  for (int e = 0; e < kRun; ++e) sum += kept(x[e], P.id(group, lane, e));
  u64 run = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 y = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += y;
  }
  if (left < run && left >= run - sum) {  // one lane
    left -= run - sum;
#pragma unroll
    for (int e = 0; e < kRun; ++e) {
      const u64 y = kept(x[e], P.id(group, lane, e));
      if (left < y) {
        out[row] = (int32_t)P.id(group, lane, e);
        break;
      }
      left -= y;
    }
  }
}

const char* sample_rows(const void* logits, int type, int64_t ld, int rows, int vocab, const float* temperature,
                        const int32_t* top_k, const float* top_p, const float* min_p, const float* uniform,
                        int32_t* out_ids, const Waits& waits, int dev, cudaStream_t st) {
  // CTAs of a row: as few as can hold it (up to 128 KB each: one CTA per SM), and more while that
  // leaves SMs idle; measured at 256 x 50257 bf16 ids without truncation: 1 CTA a row 35 us, 4 CTAs 71 us
  const int64_t bytes = (int64_t)vocab * (type == LLAMA_F32 ? 4 : 2);
  int ranks = 1;
  while (ranks < kMaxCluster && (bytes > 131000 * (int64_t)ranks || rows * ranks < 148)) ranks *= 2;
  auto launch = [&](auto x, auto r) -> const char* {
    using T = decltype(x);
    constexpr int R = decltype(r)::value;
    const int seg = (vocab + R - 1) / R;
    // a part and the slots before it, in whole groups for every warp
    const int groups = (int)(((int64_t)(seg + Part<T>::kRun) * sizeof(T) + 512 * kWarps - 1) / (512 * kWarps));
    const int smem = kSharedBytes + groups * kWarps * 512;
    if (!allow_smem(k_sample_rows<R, T>, 224 * 1024, dev)) return "shared memory could not be set";
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(rows * R));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)R;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return error_text(cudaLaunchKernelEx(&cfg, k_sample_rows<R, T>, static_cast<const T*>(logits), ld, vocab, seg, groups,
                                         temperature, top_k, top_p, min_p, uniform, out_ids, waits));
  };
  auto by_ranks = [&](auto x) {
    switch (ranks) {
      case 1: return launch(x, std::integral_constant<int, 1>{});
      case 2: return launch(x, std::integral_constant<int, 2>{});
      case 4: return launch(x, std::integral_constant<int, 4>{});
      default: return launch(x, std::integral_constant<int, 8>{});
    }
  };
  return type == LLAMA_F32 ? by_ranks(0.0f) : type == LLAMA_F16 ? by_ranks(__half{}) : by_ranks(__nv_bfloat16{});
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
  const char* why = sample_rows(logits, type, ld, rows, vocab, temperature, top_k, top_p, min_p, uniform, out_ids, Waits(),
                                dev, static_cast<cudaStream_t>(stream));
  return why ? refuse(why) : 0;
}
