// Shared parts of the paged-cache kernels: the cache as they see it, element access, a sequence's
// rows and keys, and the joining of key splits.
//
// The cache is a pool of pages of page_size rows; sequence s keeps key j in row j % page_size of
// page table[s][j / page_size].  A page id outside [0, num_pages) holds no rows: nothing is
// written there and its keys are left out of the softmax, so that a bad table cannot send an
// access out of the pool.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace le {
namespace paged {

// What the kernels need of llama_paged_kv_t.
struct Cache {
  void* k;
  void* v;
  const int32_t* table;
  const int32_t* slots;  // row of the table of each sequence, or nullptr: the sequence's own number
  int64_t page_stride, row_stride, head_stride;  // elements
  int table_stride, table_width, table_rows, seqs, num_pages, page_log2, kv_heads;
};

template <typename T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32(float x) { return x; }
template <> __device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float x) { return __float2bfloat16_rn(x); }

// 8 consecutive elements, 16-byte accesses (two for fp32).
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(e[i]);
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    uint4 u;
    T* e = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(x[i]);
    *reinterpret_cast<uint4*>(p) = u;
  }
}

// The page ids of sequence s (nullptr: a slot outside the table, whose keys do not exist).
__device__ __forceinline__ const int32_t* pages_of(const Cache& C, int s) {
  const int row = C.slots ? C.slots[s] : s;
  return row >= 0 && row < C.table_rows ? C.table + (int64_t)row * C.table_stride : nullptr;
}
// Page of entry e, or -1 where there is none.
__device__ __forceinline__ int page_at(const Cache& C, const int32_t* pages, int e) {
  const int p = pages && e < C.table_width ? pages[e] : -1;
  return p < C.num_pages ? p : -1;
}
// Row of key j in the pools (element offset of kv head g), or -1.
__device__ __forceinline__ int64_t key_offset(const Cache& C, const int32_t* pages, int j, int g) {
  const int page = page_at(C, pages, j >> C.page_log2);
  if (page < 0) return -1;
  return (int64_t)page * C.page_stride + (int64_t)(j & ((1 << C.page_log2) - 1)) * C.row_stride +
         (int64_t)g * C.head_stride;
}

// Two fp32 values rounded to T, the first in the low half.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// 2^x (ex2.approx: 2^-22 relative; 2^-inf = 0).
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Rows and keys of sequence s.  Rows outside [0, rows) and keys past the table do not exist.
struct Span {
  int first, n, len;  // first row, rows, keys
};
__device__ __forceinline__ Span span_of(const Cache& C, const int32_t* cu_q, const int32_t* kv_len, int s, int rows) {
  Span x;
  const int a = cu_q[s], b = cu_q[s + 1];
  x.first = max(a, 0);
  x.n = min(b, rows) - x.first;
  // clipping only keeps accesses in range: the callers' rows end at cu_q[seqs] <= rows
  x.len = max(0, min(kv_len[s], C.table_width << C.page_log2));
  return x;
}

// Key splits that a sequence of len keys is cut into (at least one, which writes the zeros of a
// sequence without keys).
__host__ __device__ __forceinline__ int splits_of(int len, int per, int splits) {
  const int u = (len + per - 1) / per;
  return u < 1 ? 1 : u > splits ? splits : u;
}

// A split's part of a (row, head): D unnormalised outputs, then the maximum (log2 units) and sum.
template <int D>
__device__ __forceinline__ void write_part(float* part, int64_t index, int d, float m, float l, const float (&a)[8]) {
  float* p = part + index * (D + 8);
  store8(p + d, a);
  if (d == 0) *reinterpret_cast<float2*>(p + D) = make_float2(m, l);
}

// How the keys are split and where the parts lie.  [0]: sequences of at most small_rows query rows
// per kv head, their parts by (sequence, kv head, row of the tile); [1]: the others, by (row, head),
// behind part1 parts of the first kind.
constexpr int kDecodeRows = 16;  // query rows of a decode tile: G heads x new tokens
struct SplitPlan {
  int per[2], splits[2], small_rows;
  int64_t part1;
};

// out = sum_z 2^(m_z - M) o_z / sum_z 2^(m_z - M) l_z over the splits of a (row, head), M = max m_z;
// rows whose sequence has one split were written already.  The first blocks0 blocks take the rows of
// decode tiles (tile_rows of each sequence and kv head), the others all rows, of which those of chunks are
// theirs.  D / 8 << groups_log2 threads per (row, head), 8 outputs each: a group of D / 8 takes every
// groups-th split with a running (M, L, o), and the groups join through shared memory.  A thread's loads
// follow one another's addresses only, so kCombineRun splits are in flight at a time.  Against one group
// that walks all splits: attention of one token, 8 kv heads of 64, over 32768 keys (64 splits) 26.5 -> 17.9
// us, over 4096 (22) 10.7 -> 7.8 us.  Against looking every row of the call up: 32 chunks of 256 over 4096, with a single
// token and an idle sequence among them, 279 -> 216 us.
constexpr int kCombineThreads = 128, kCombineRun = 4;
template <typename O, int D>
__global__ void __launch_bounds__(kCombineThreads)
    k_paged_combine(Cache C, int heads, const int32_t* __restrict__ cu_q, const int32_t* __restrict__ kv_len, int rows,
                    SplitPlan P, int blocks0, int tile_rows, int groups_log2, const float* __restrict__ part,
                    O* __restrict__ out, int64_t out_ld) {
  grid_dep_wait();  // the parts come from the kernel before
  constexpr int kRuns = D / 8;
  __shared__ __align__(16) float s_a[kCombineThreads][8];
  __shared__ float2 s_ml[kCombineThreads];
  const int groups = 1 << groups_log2, mine = threadIdx.x % kRuns, grp = threadIdx.x / kRuns % groups;
  const int d = mine * 8, G = heads / C.kv_heads;
  int used = 0, t = 0, h = 0;  // splits to join: none where the row is nobody's, or has been written
  const float* p = part;
  if ((int)blockIdx.x < blocks0) {
    const int64_t i = ((int64_t)blockIdx.x * kCombineThreads + threadIdx.x) / (kRuns * groups);
    const int r = (int)(i % tile_rows), g = (int)(i / tile_rows % C.kv_heads);
    const int64_t s = i / tile_rows / C.kv_heads;
    if (s < C.seqs) {
      const Span sp = span_of(C, cu_q, kv_len, (int)s, rows);
      t = sp.first + r / G;
      h = g * G + r % G;
      if (r < sp.n * G && sp.n * G <= P.small_rows) used = splits_of(sp.len, P.per[0], P.splits[0]);
      if (used > 1) p += ((s * C.kv_heads + g) * kDecodeRows + r) * P.splits[0] * (D + 8);
    }
  } else {
    const int64_t rh = ((int64_t)(blockIdx.x - blocks0) * kCombineThreads + threadIdx.x) / (kRuns * groups);
    t = (int)(rh / heads);
    h = (int)(rh % heads);
    if (t < rows) {
      int lo = 0, hi = C.seqs;  // sequence of row t: the first whose end lies behind it
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (cu_q[mid + 1] <= t) lo = mid + 1;
        else hi = mid;
      }
      if (lo < C.seqs) {
        const Span sp = span_of(C, cu_q, kv_len, lo, rows);
        if (t >= sp.first && sp.n * G > P.small_rows) used = splits_of(sp.len, P.per[1], P.splits[1]);
        if (used > 1) p += (P.part1 + rh * P.splits[1]) * (D + 8);
      }
    }
  }
  float M = -INFINITY, L = 0.0f, a[8] = {};
  auto join = [&](float2 ml, const float (&x)[8]) {
    const float m = fmaxf(M, ml.x);
    const float f = ml.x == -INFINITY ? 0.0f : exp2_approx(ml.x - m), g = M == -INFINITY ? 0.0f : exp2_approx(M - m);
    M = m;
    L = fmaf(ml.y, f, L * g);
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e] = fmaf(x[e], f, a[e] * g);
  };
  if (used > 1) {
    for (int z0 = grp; z0 < used; z0 += kCombineRun * groups) {
      float2 ml[kCombineRun];
      float x[kCombineRun][8];
#pragma unroll
      for (int i = 0; i < kCombineRun; ++i) {
        const float* pz = p + (int64_t)min(z0 + i * groups, used - 1) * (D + 8);
        ml[i] = *reinterpret_cast<const float2*>(pz + D);
        load8(pz + d, x[i]);
      }
#pragma unroll
      for (int i = 0; i < kCombineRun; ++i)
        if (z0 + i * groups < used) join(ml[i], x[i]);
    }
  }
  if (groups > 1) {  // the block's own (row, head)s: all threads come here
    store8(s_a[threadIdx.x], a);
    s_ml[threadIdx.x] = make_float2(M, L);
    __syncthreads();
    if (grp) return;
    for (int y = 1; y < groups; ++y) {
      float x[8];
      load8(s_a[threadIdx.x + y * kRuns], x);
      join(s_ml[threadIdx.x + y * kRuns], x);
    }
  }
  if (used <= 1) return;
  const float inv = L > 0.0f ? 1.0f / L : L == L ? 0.0f : L;  // no key: zeros
#pragma unroll
  for (int e = 0; e < 8; ++e) a[e] *= inv;
  store8(out + (int64_t)t * out_ld + (int64_t)h * D + d, a);
}

}  // namespace paged
}  // namespace le
