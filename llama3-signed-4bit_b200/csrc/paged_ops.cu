// Paged KV cache operators behind the C ABI: llama_paged_append (RoPE and append) and
// llama_paged_attention (attention of new tokens over the cache).
//
// The cache is a pool of pages of page_size rows; sequence s keeps key j in row j % page_size of
// page table[s][j / page_size].  A page id outside [0, num_pages) holds no rows: nothing is
// written there and its keys are left out of the softmax, so that a bad table cannot send an
// access out of the pool.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "ops.h"

#define LE_API extern "C" __attribute__((visibility("default")))

namespace le {
namespace paged {

// What the kernels need of llama_paged_kv_t.
struct Cache {
  void* k;
  void* v;
  const int32_t* table;
  int64_t page_stride, row_stride, head_stride;  // elements
  int table_stride, table_width, seqs, num_pages, page_log2, kv_heads;
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

// Row of key j of sequence s in the pools (element offset of kv head g), or -1 when the table
// holds no valid page for it.
__device__ __forceinline__ int64_t key_offset(const Cache& C, int s, int j, int g) {
  const int i = j >> C.page_log2;
  if (i >= C.table_width) return -1;
  const int page = C.table[(int64_t)s * C.table_stride + i];
  if (page < 0 || page >= C.num_pages) return -1;
  return (int64_t)page * C.page_stride + (int64_t)(j & ((1 << C.page_log2) - 1)) * C.row_stride +
         (int64_t)g * C.head_stride;
}

// ---------------------------------------------------------------------------------------------
// Append.  Row t of qkv is q heads | k heads | v heads; with (c, s) the table row of its position,
// rot(x)_i = x_i c_i - x_{i + D/2} s_i and rot(x)_{i + D/2} = x_i s_i + x_{i + D/2} c_i for
// i < D/2, in fp32 without contraction (the engine's own rotation), rounded once to the output
// type.  A thread takes 8 rotation pairs of one head: two 16-byte runs half a head apart.
// ---------------------------------------------------------------------------------------------
template <typename In, typename Kv, typename Q, int D>
__global__ void __launch_bounds__(256)
    k_paged_append(Cache C, const In* __restrict__ qkv, int64_t ld, int rows, int heads,
                   const int32_t* __restrict__ pos, const int32_t* __restrict__ seq,
                   const float* __restrict__ rope_cos, const float* __restrict__ rope_sin, int n_pos,
                   Q* __restrict__ q_out, int64_t q_ld) {
  constexpr int kRuns = D / 16;
  const int per_row = (heads + 2 * C.kv_heads) * kRuns;
  const int64_t item = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (item >= (int64_t)rows * per_row) return;
  const int t = (int)(item / per_row);
  const int r = (int)(item - (int64_t)t * per_row);
  const int h = r / kRuns, i0 = (r % kRuns) * 8;
  const int p = pos[t], s = seq[t];
  if (s < 0 || s >= C.seqs || p < 0 || p >= n_pos) return;  // a row of no sequence
  const In* src = qkv + (int64_t)t * ld + (int64_t)h * D + i0;
  float a[8], b[8];
  load8(src, a);
  load8(src + D / 2, b);
  if (h < heads + C.kv_heads) {
    float c[8], sn[8];
    load8(rope_cos + (int64_t)p * (D / 2) + i0, c);
    load8(rope_sin + (int64_t)p * (D / 2) + i0, sn);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = a[i], y = b[i];
      a[i] = __fsub_rn(__fmul_rn(x, c[i]), __fmul_rn(y, sn[i]));
      b[i] = __fadd_rn(__fmul_rn(x, sn[i]), __fmul_rn(y, c[i]));
    }
  }
  if (h < heads) {
    Q* dst = q_out + (int64_t)t * q_ld + (int64_t)h * D + i0;
    store8(dst, a);
    store8(dst + D / 2, b);
    return;
  }
  const bool is_k = h < heads + C.kv_heads;
  const int64_t off = key_offset(C, s, p, is_k ? h - heads : h - heads - C.kv_heads);
  if (off < 0) return;
  Kv* dst = static_cast<Kv*>(is_k ? C.k : C.v) + off + i0;
  store8(dst, a);
  store8(dst + D / 2, b);
}

// ---------------------------------------------------------------------------------------------
// Attention: o = sum_j p_j v_j with p = softmax(scale q . k_j) over the keys 0 .. position of the
// token, one pass with a running maximum and sum (fp32).  One warp per (token, head).
// ---------------------------------------------------------------------------------------------
template <typename T, typename O, int D>
__global__ void __launch_bounds__(128)
    k_paged_attention(Cache C, const T* __restrict__ q, int64_t q_ld, int heads, const int32_t* __restrict__ cu_q,
                      const int32_t* __restrict__ kv_len, int rows, float scale, O* __restrict__ out, int64_t out_ld) {
  constexpr int kE = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t w = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (w >= (int64_t)rows * heads) return;
  const int t = (int)(w / heads), h = (int)(w % heads);
  int lo = 0, hi = C.seqs;  // sequence of row t: cu_q[lo] <= t < cu_q[lo + 1]
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cu_q[mid + 1] <= t) lo = mid + 1;
    else hi = mid;
  }
  if (lo >= C.seqs || t < cu_q[lo]) return;  // a row behind the last sequence
  const int s = lo, g = h / (heads / C.kv_heads);
  const int last = min(kv_len[s], C.table_width << C.page_log2) - (cu_q[s + 1] - t);
  float qv[kE], o[kE], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int e = 0; e < kE; ++e) {
    qv[e] = to_f32(q[(int64_t)t * q_ld + (int64_t)h * D + lane * kE + e]) * scale;
    o[e] = 0.0f;
  }
  for (int j = 0; j <= last; ++j) {
    const int64_t off = key_offset(C, s, j, g);
    if (off < 0) continue;
    const T* kr = static_cast<const T*>(C.k) + off + lane * kE;
    const T* vr = static_cast<const T*>(C.v) + off + lane * kE;
    float d = 0.0f;
#pragma unroll
    for (int e = 0; e < kE; ++e) d = fmaf(qv[e], to_f32(kr[e]), d);
    d = warp_sum(d);
    if (d == -INFINITY) continue;
    const float mn = fmaxf(m, d);
    const float alpha = expf(m - mn), p = expf(d - mn);
    l = l * alpha + p;
    m = mn;
#pragma unroll
    for (int e = 0; e < kE; ++e) o[e] = fmaf(o[e], alpha, p * to_f32(vr[e]));
  }
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;  // no key: zeros
#pragma unroll
  for (int e = 0; e < kE; ++e) out[(int64_t)t * out_ld + (int64_t)h * D + lane * kE + e] = from_f32<O>(o[e] * inv);
}

static int refuse(const char* what, const char* why, int rc = -1) {
  set_global_error(std::string(what) + ": " + why);
  return rc;
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
static int type_size(int t) { return t == LLAMA_F32 ? 4 : 2; }

// Checks a cache descriptor; the reason of a refusal, or nullptr.
static const char* check_cache(const llama_paged_kv_t* kv) {
  if (!kv) return "cache descriptor is NULL";
  if (!kv->k || !kv->v || !kv->table) return "cache descriptor holds a NULL pointer";
  if (kv->type != LLAMA_F16 && kv->type != LLAMA_BF16) return "cache type must be LLAMA_F16 or LLAMA_BF16";
  if (kv->head_dim != 64 && kv->head_dim != 128) return "head_dim must be 64 or 128";
  if (kv->page_size < 16 || kv->page_size > 256 || (kv->page_size & (kv->page_size - 1)) != 0)
    return "page_size must be 16, 32, 64, 128 or 256";
  if (kv->num_pages < 1 || kv->kv_heads < 1 || kv->seqs < 1) return "num_pages, kv_heads and seqs must be positive";
  if (kv->table_width < 1 || kv->table_stride < kv->table_width) return "table_stride must be at least table_width >= 1";
  if (kv->table_width > (1 << 30) / kv->page_size) return "table_width is too large";
  if (!aligned16(kv->k) || !aligned16(kv->v)) return "k and v must be 16-byte aligned";
  const int64_t st[3] = {kv->page_stride, kv->row_stride, kv->head_stride};
  for (int64_t x : st)
    if (x < kv->head_dim || x % 8 != 0 || x >= ((int64_t)1 << 38)) return "strides must be multiples of 8 elements, at least head_dim";
  return nullptr;
}

static Cache cache_of(const llama_paged_kv_t* kv) {
  Cache c{};
  c.k = kv->k;
  c.v = kv->v;
  c.table = kv->table;
  c.page_stride = kv->page_stride;
  c.row_stride = kv->row_stride;
  c.head_stride = kv->head_stride;
  c.table_stride = kv->table_stride;
  c.table_width = kv->table_width;
  c.seqs = kv->seqs;
  c.num_pages = kv->num_pages;
  while ((1 << c.page_log2) < kv->page_size) ++c.page_log2;
  c.kv_heads = kv->kv_heads;
  return c;
}

}  // namespace paged
}  // namespace le

using namespace le;

LE_API int llama_paged_append(const llama_paged_kv_t* kv, const void* qkv, int type, int64_t ld, int rows, int heads,
                              const int32_t* pos, const int32_t* seq, const float* rope_cos, const float* rope_sin,
                              int n_pos, void* q_out, int q_type, int64_t q_ld, void* stream) {
  using namespace paged;
  const char* who = "llama_paged_append";
  if (const char* why = check_cache(kv)) return refuse(who, why);
  if (!qkv || !pos || !seq || !rope_cos || !rope_sin || !q_out) return refuse(who, "NULL argument");
  if (type != LLAMA_F32 && type != kv->type) return refuse(who, "type must be LLAMA_F32 or the cache's type");
  if (q_type != type && q_type != kv->type) return refuse(who, "q_type must be the input's or the cache's type");
  if (rows < 0 || n_pos < 1) return refuse(who, "rows and n_pos out of range");
  if (heads < 1 || heads > 4096 || heads % kv->kv_heads != 0) return refuse(who, "heads must be a multiple of kv_heads");
  const int D = kv->head_dim;
  if (ld < (int64_t)(heads + 2 * kv->kv_heads) * D || (ld * type_size(type)) % 16 != 0)
    return refuse(who, "ld is shorter than a row or not a multiple of 16 bytes");
  if (q_ld < (int64_t)heads * D || (q_ld * type_size(q_type)) % 16 != 0)
    return refuse(who, "q_ld is shorter than a row or not a multiple of 16 bytes");
  if (!aligned16(qkv) || !aligned16(q_out) || !aligned16(rope_cos) || !aligned16(rope_sin))
    return refuse(who, "qkv, q_out and the RoPE tables must be 16-byte aligned");
  if (rows == 0) return 0;
  const int dev = device_of(kv->k);
  const void* ptrs[] = {kv->v, kv->table, qkv, pos, seq, rope_cos, rope_sin, q_out};
  for (const void* p : ptrs)
    if (dev < 0 || device_of(p) != dev) return refuse(who, "every pointer must be memory of one CUDA device");
  DeviceGuard dg(dev);
  const Cache C = cache_of(kv);
  const int64_t items = (int64_t)rows * (heads + 2 * kv->kv_heads) * (D / 16);
  if (items > (int64_t)256 * 0x7fffffff) return refuse(who, "rows out of range");
  const unsigned grid = (unsigned)((items + 255) / 256);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto launch = [&](auto in, auto c, auto q) {
    using In = decltype(in);
    using Kv = decltype(c);
    using Q = decltype(q);
    auto* fn = D == 64 ? k_paged_append<In, Kv, Q, 64> : k_paged_append<In, Kv, Q, 128>;
    fn<<<grid, 256, 0, st>>>(C, static_cast<const In*>(qkv), ld, rows, heads, pos, seq, rope_cos, rope_sin, n_pos,
                             static_cast<Q*>(q_out), q_ld);
  };
  auto by_type = [&](auto c) {
    if (type != LLAMA_F32) launch(c, c, c);
    else if (q_type == LLAMA_F32) launch(0.0f, c, 0.0f);
    else launch(0.0f, c, c);
  };
  if (kv->type == LLAMA_F16) by_type(__half{});
  else by_type(__nv_bfloat16{});
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : refuse(who, cudaGetErrorString(e));
}

LE_API size_t llama_paged_attention_workspace(const llama_paged_kv_t* kv, int heads, int rows, int max_q, int max_kv) {
  (void)heads; (void)rows; (void)max_q; (void)max_kv;
  return paged::check_cache(kv) ? 0 : 16;
}

LE_API int llama_paged_attention(const llama_paged_kv_t* kv, const void* q, int64_t q_ld, int heads,
                                 const int32_t* cu_q, const int32_t* kv_len, int rows, int max_q, int max_kv,
                                 float scale, void* out, int out_type, int64_t out_ld, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  using namespace paged;
  const char* who = "llama_paged_attention";
  if (const char* why = check_cache(kv)) return refuse(who, why);
  if (!q || !cu_q || !kv_len || !out) return refuse(who, "NULL argument");
  if (out_type != LLAMA_F32 && out_type != kv->type) return refuse(who, "out_type must be LLAMA_F32 or the cache's type");
  if (rows < 0 || max_q < 0 || max_kv < 0) return refuse(who, "rows, max_q and max_kv must not be negative");
  if (heads < 1 || heads > 4096 || heads % kv->kv_heads != 0) return refuse(who, "heads must be a multiple of kv_heads");
  if (!(std::fabs(scale) <= 3.0e38f)) return refuse(who, "scale must be finite");
  const int D = kv->head_dim;
  if (q_ld < (int64_t)heads * D || q_ld % 8 != 0) return refuse(who, "q_ld is shorter than a row or not a multiple of 8");
  if (out_ld < (int64_t)heads * D || out_ld % 8 != 0) return refuse(who, "out_ld is shorter than a row or not a multiple of 8");
  if (!aligned16(q) || !aligned16(out)) return refuse(who, "q and out must be 16-byte aligned");
  const size_t need = llama_paged_attention_workspace(kv, heads, rows, max_q, max_kv);
  if (need > 16 && (!workspace || !aligned16(workspace) || workspace_bytes < need))
    return refuse(who, "workspace is too small", -2);
  if (rows == 0) return 0;
  const int dev = device_of(kv->k);
  const void* ptrs[] = {kv->v, kv->table, q, cu_q, kv_len, out};
  for (const void* p : ptrs)
    if (dev < 0 || device_of(p) != dev) return refuse(who, "every pointer must be memory of one CUDA device");
  DeviceGuard dg(dev);
  const Cache C = cache_of(kv);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const unsigned grid = (unsigned)(((int64_t)rows * heads + 3) / 4);
  auto launch = [&](auto c, auto o) {
    using T = decltype(c);
    using O = decltype(o);
    auto* fn = D == 64 ? k_paged_attention<T, O, 64> : k_paged_attention<T, O, 128>;
    fn<<<grid, 128, 0, st>>>(C, static_cast<const T*>(q), q_ld, heads, cu_q, kv_len, rows, scale, static_cast<O*>(out),
                             out_ld);
  };
  auto by_type = [&](auto c) {
    if (out_type == LLAMA_F32) launch(c, 0.0f);
    else launch(c, c);
  };
  if (kv->type == LLAMA_F16) by_type(__half{});
  else by_type(__nv_bfloat16{});
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : refuse(who, cudaGetErrorString(e));
}
