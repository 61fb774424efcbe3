// Paged KV cache operators behind the C ABI: llama_paged_append (RoPE and append) and
// llama_paged_attention (attention of new tokens over the cache).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "ops.h"
#include "paged.cuh"
#include "paged_chunk.cuh"
#include "paged_decode.cuh"

#define LE_API extern "C" __attribute__((visibility("default")))

namespace le {
namespace paged {

// ---------------------------------------------------------------------------------------------
// Append.  Row t of qkv is q heads | k heads | v heads; with (c, s) the table row of its position,
// rot(x)_i = x_i c_i - x_{i + D/2} s_i and rot(x)_{i + D/2} = x_i s_i + x_{i + D/2} c_i for
// i < D/2, in fp32 without contraction (the engine's own rotation), rounded once to the output
// type.  A thread takes 8 rotation pairs of one head: two 16-byte runs half a head apart.  With
// planes > 1 (the engine's split-K products, fp32) a row is the sum of its planes, in plane order.
//
// Bound by its bytes for chunks, by the launch and three loads in a row (position, page, data) for decode
// steps.  8192 rows of 32 + 8 + 8 heads of 64, fp32 to fp16: 30.5 us (153 MB, 5.0 TB/s); 2048 rows:
// 7.1 us; 64 rows: 2.7 us.  Threads that take 4 heads and load their cosines once: 30.7, 8.1 and
// 2.7 us, since L1 serves the cosines of a row's heads.
// ---------------------------------------------------------------------------------------------
template <typename In, typename Kv, typename Q, int D>
__global__ void __launch_bounds__(256)
    k_paged_append(Cache C, const In* __restrict__ qkv, int64_t ld, int planes, int64_t plane_stride, int rows, int heads,
                   const int32_t* __restrict__ pos, const int32_t* __restrict__ seq,
                   const float* __restrict__ rope_cos, const float* __restrict__ rope_sin, int n_pos,
                   Q* __restrict__ q_out, int64_t q_ld) {
  constexpr int kRuns = D / 16;
  grid_dep_begin();
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
  for (int j = 1; j < planes; ++j) {
    float x[8], y[8];
    load8(src + j * plane_stride, x);
    load8(src + j * plane_stride + D / 2, y);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a[i] += x[i];
      b[i] += y[i];
    }
  }
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
  const int64_t off = key_offset(C, pages_of(C, s), p, is_k ? h - heads : h - heads - C.kv_heads);
  if (off < 0) return;
  Kv* dst = static_cast<Kv*>(is_k ? C.k : C.v) + off + i0;
  store8(dst, a);
  store8(dst + D / 2, b);
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
  if (kv->slots ? kv->table_rows < 1 : kv->table_rows != 0) return "table_rows must be positive with slots, 0 without";
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
  c.slots = kv->slots;
  c.table_rows = kv->slots ? kv->table_rows : kv->seqs;
  c.seqs = kv->seqs;
  c.num_pages = kv->num_pages;
  while ((1 << c.page_log2) < kv->page_size) ++c.page_log2;
  c.kv_heads = kv->kv_heads;
  return c;
}

// A launch that may start while the kernel before it runs out; that kernel's results are there
// after its griddepcontrol.wait.  nullptr, or why it failed (an earlier call's error is not looked at).
template <typename... KArgs, typename... Args>
static const char* launch(bool early, void (*kernel)(KArgs...), unsigned grid, unsigned block, size_t smem, cudaStream_t s,
                   int cluster, Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  cfg.attrs = at;
  if (early) {
    at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    at[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    at[cfg.numAttrs].val.clusterDim.x = (unsigned)cluster;
    at[cfg.numAttrs].val.clusterDim.y = at[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  return error_text(cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...));
}

const char* append_rows(const llama_paged_kv_t* kv, const void* qkv, int type, int64_t ld, int planes,
                        int64_t plane_stride, int rows, int heads, const int32_t* pos, const int32_t* seq,
                        const float* rope_cos, const float* rope_sin, int n_pos, void* q_out, int q_type, int64_t q_ld,
                        cudaStream_t st, bool chained) {
  const Cache C = cache_of(kv);
  const int D = kv->head_dim;
  const int64_t items = (int64_t)rows * (heads + 2 * kv->kv_heads) * (D / 16);
  if (items > (int64_t)256 * 0x7fffffff) return "rows out of range";
  const unsigned grid = (unsigned)((items + 255) / 256);
  auto run = [&](auto in, auto c, auto q) {
    using In = decltype(in);
    using Kv = decltype(c);
    using Q = decltype(q);
    auto* fn = D == 64 ? k_paged_append<In, Kv, Q, 64> : k_paged_append<In, Kv, Q, 128>;
    return launch(chained, fn, grid, 256, 0, st, 1, C, static_cast<const In*>(qkv), ld, planes, plane_stride, rows, heads, pos,
                  seq, rope_cos, rope_sin, n_pos, static_cast<Q*>(q_out), q_ld);
  };
  auto by_type = [&](auto c) {
    return type != LLAMA_F32 ? run(c, c, c) : q_type == LLAMA_F32 ? run(0.0f, c, 0.0f) : run(0.0f, c, c);
  };
  return kv->type == LLAMA_F16 ? by_type(__half{}) : by_type(__nv_bfloat16{});
}

constexpr int kSms = 148;  // the workspace's size must not need a device
constexpr int kSmSharedBytes = 227 * 1024;  // that an SM's CTAs can have together
constexpr int kChunkItems = 4 * kSms;  // bounds what splitting makes
constexpr double kKeysRoot = 0.9;
constexpr int kIdleItems = 8192;  // decode CTAs of a call with more sequences than rows
constexpr int kLongestBytes = 640 << 20;  // of keys and values when all have max_kv of them; L2 has 126 MB

// How a call is cut: which kernels run, and their key splits.
struct Plan {
  SplitPlan sp{};
  bool decode = false, chunk = false, join = false;  // join: decode splits are joined by clusters
  bool longest = false;  // chunk items in order of their keys
  size_t bytes = 0;
};
static Plan plan_of(const llama_paged_kv_t* kv, int heads, int rows, int max_q, int max_kv) {
  Plan P;
  const int G = heads / kv->kv_heads;
  const int64_t keys = std::max<int64_t>(1, std::min<int64_t>(max_kv, (int64_t)kv->table_width * kv->page_size));
  P.chunk = (int64_t)max_q * G > kDecodeRows;
  // beside chunks there are sequences of few tokens unless all have max_q of them
  P.decode = !P.chunk || (kv->seqs > 1 && rows < (int64_t)kv->seqs * max_q && G <= kDecodeRows);
  P.sp.small_rows = P.decode ? kDecodeRows : 0;
  const int64_t units = (int64_t)std::min(kv->seqs, std::max(rows, 1)) * kv->kv_heads;
  // decode: a CTA's start and end cost as much as some hundred keys, and the last CTAs of many short ones
  // end closer together, so keys per CTA and CTAs grow alike, as the root of the call's keys.  At 0.9 of
  // it 64 x 2048 takes 34.6 us (0.7, with a quarter more parts in memory: 34.0; 1.4: 35.7), 128 x 8192 319
  // us (313, 329), 1 x 4096 7.8 us (7.5, 9.0), 1 x 32768 17.9 us (17.5, 16.2); 128 keys are two slices for
  // each warp.
  auto whole = [](int64_t n) { return std::max<int64_t>(128, (n + 63) / 64 * 64); };
  auto keys_each = [&](int64_t of) {
    return std::min(whole((int64_t)std::ceil(kKeysRoot * std::sqrt((double)of * keys))), whole(keys));
  };
  int64_t per = keys_each(units);
  int64_t parts = (keys + per - 1) / per;
  // Described sequences without a row launch as many CTAs and have room for as many parts as the others, so
  // their number bounds the splits: one row over 8192 keys among 256 sequences (8 kv heads of 128) took 121 us
  // and 570 MB for 32 splits, which it has alone.
  const int64_t all = (int64_t)kv->seqs * kv->kv_heads;
  if (all > units) {
    const int64_t root = keys_each(all), most = std::max<int64_t>(kIdleItems / all, (keys + root - 1) / root);
    if (parts > most) {
      per = whole((keys + most - 1) / most);
      parts = (keys + per - 1) / per;
    }
  }
  // Where all CTAs can be resident at once, a cluster of them takes each pair and joins its splits: no second
  // launch, no parts in memory, and every sequence cut evenly (1 x 700 9.2 -> 6.1 us, 16 x 2048 13.6 -> 12.7,
  // 8 x 2048 with heads of 128 19.0 -> 15.0).  Beyond that clusters wait for one another's shared memory (64 x
  // 2048, clusters of 4: 36 -> 44 us), and pairs whose keys are worth many more CTAs than a cluster has
  // are faster without (1 x 32768, clusters of 8: 18.5 -> 35 us).
  const int64_t resident = (int64_t)kSms * (kSmSharedBytes / (kv->head_dim == 64 ? DecodeGeo<64>::kSmem : DecodeGeo<128>::kSmem));
  const int64_t joined = std::min({(int64_t)kJoinSplits, resident / units, (keys + kJoinKeys - 1) / kJoinKeys});
  P.join = P.decode && joined > 1 && parts <= 2 * kJoinSplits;
  if (P.join) parts = joined;
  P.sp.per[0] = (int)per;
  P.sp.splits[0] = P.decode ? (int)parts : 1;
  // chunk: one CTA per SM; as many splits as make the estimate smallest: the busiest SM's key tiles,
  // three more for each of its items, and the parts' way through memory, of which about 8 MB pass in the
  // 1.9 us of a key tile.  512 tokens over 32768 keys (8 x 8 items): 2 splits 251 us, 9 (which would
  // fill the SMs better) 290 us.
  P.sp.per[1] = 1 << 30;
  P.sp.splits[1] = 1;
  if (P.chunk) {
    const RowTiles R = row_tiles(G);
    const int64_t tiles = ((int64_t)rows + R.tokens - 1) / R.tokens * R.parts;
    const int64_t items = std::max<int64_t>(1, (tiles + 1) / 2) * kv->kv_heads;
    const double part_tiles = (double)rows * heads * (kv->head_dim + 8) * 8 / 8e6;
    double best = -1;
    for (int64_t n = 1; n == 1 || (n <= 32 && keys >= 512 * n && items * n <= kChunkItems); ++n) {
      const int64_t p1 = (keys + n * kTileKeys - 1) / (n * kTileKeys) * kTileKeys;
      const double cost = (double)((items * n + kSms - 1) / kSms) * (p1 / kTileKeys + 3) + (n > 1 ? 2 + n * part_tiles : 0);
      if (best < 0 || cost < best) {
        best = cost;
        P.sp.per[1] = n == 1 ? 1 << 30 : (int)p1;
        P.sp.splits[1] = (int)((keys + p1 - 1) / p1);
      }
    }
    // The longest items first where SMs take several: 8 ragged chunks of 611 over 3001 104 -> 94 us.  Not
    // where the sequences' keys are far beyond L2, since each item then brings its own from memory: 16
    // equal chunks of 1024 over 16384 take 3.53 -> 3.82 ms so.  Up to 32 sequences, a lane each; with four
    // for each lane every look-up takes longer than the order gains (8 x 2048 248 -> 250 us).
    P.longest = kv->seqs > 1 && kv->seqs <= 32 && items * P.sp.splits[1] > kSms &&
                units * keys * kv->head_dim * 4 <= (int64_t)kLongestBytes;
  }
  const int64_t n0 = P.sp.splits[0] > 1 && !P.join ? (int64_t)kv->seqs * kv->kv_heads * kDecodeRows * P.sp.splits[0] : 0;
  const int64_t n1 = P.sp.splits[1] > 1 ? (int64_t)rows * heads * P.sp.splits[1] : 0;
  P.sp.part1 = n0;
  P.bytes = (size_t)(n0 + n1) * (kv->head_dim + 8) * sizeof(float);
  return P;
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
// A TMA map of 16-bit elements with 128-byte swizzle; what lies outside reads as zeros.
static bool make_map(CUtensorMap* m, int type, int rank, const void* at, const cuuint64_t* dims, const cuuint64_t* strides,
                     const cuuint32_t* box) {
  static const EncodeTiled encode = [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult st;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &st) != cudaSuccess) fn = nullptr;
    return reinterpret_cast<EncodeTiled>(fn);
  }();
  const cuuint32_t one[4] = {1, 1, 1, 1};
  return encode &&
         encode(m, type == LLAMA_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)rank,
                const_cast<void*>(at), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// A pool as (element, head, row, page): boxes of 64 elements x one head x up to 128 rows of a page.
static bool pool_map(CUtensorMap* m, const llama_paged_kv_t* kv, const void* pool) {
  const cuuint64_t dims[4] = {(cuuint64_t)kv->head_dim, (cuuint64_t)kv->kv_heads, (cuuint64_t)kv->page_size,
                              (cuuint64_t)kv->num_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)kv->head_stride * 2, (cuuint64_t)kv->row_stride * 2,
                                 (cuuint64_t)kv->page_stride * 2};
  const cuuint32_t box[4] = {64, 1, (cuuint32_t)std::min(kv->page_size, kTileKeys), 1};
  return make_map(m, kv->type, 4, pool, dims, strides, box);
}
// The queries as (element, head, token): boxes of 64 elements x a row tile's heads x its tokens.
static bool query_map(CUtensorMap* m, const llama_paged_kv_t* kv, const void* q, int64_t q_ld, int heads, int rows) {
  const RowTiles R = row_tiles(heads / kv->kv_heads);
  const cuuint64_t dims[3] = {(cuuint64_t)kv->head_dim, (cuuint64_t)heads, (cuuint64_t)rows};
  const cuuint64_t strides[2] = {(cuuint64_t)kv->head_dim * 2, (cuuint64_t)q_ld * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)R.heads, (cuuint32_t)R.tokens};
  return make_map(m, kv->type, 3, q, dims, strides, box);
}

template <typename T, typename O, int D>
static const char* attention(const llama_paged_kv_t* kv, const Plan& P, const Cache& C, int dev, const void* q, int64_t q_ld, int heads,
                             const int32_t* cu_q, const int32_t* kv_len, int rows, int max_q, float scale, void* out,
                             int64_t out_ld, float* part, const Waits& waits, cudaStream_t st, bool chained) {
  const T* qt = static_cast<const T*>(q);
  O* ot = static_cast<O*>(out);
  if (P.chunk) {
    // two row tiles an item, every sequence's last one perhaps half empty
    const RowTiles R = row_tiles(heads / C.kv_heads);
    const int64_t pairs = ((int64_t)rows * R.parts + 2 * R.tokens - 1) / (2 * R.tokens) + std::min(C.seqs, rows);
    const int64_t items = pairs * C.kv_heads * P.sp.splits[1];
    if (items > 0x3fffffff) return "too many rows";
    CUtensorMap mq, mk, mv;
    if (!query_map(&mq, kv, q, q_ld, heads, rows) || !pool_map(&mk, kv, kv->k) || !pool_map(&mv, kv, kv->v))
      return "tensor maps could not be made";
    if (!allow_smem(k_paged_chunk<T, O, D>, ChunkGeo<D>::kSmem, dev)) return "shared memory could not be set";
    if (const char* why = launch(chained, k_paged_chunk<T, O, D>, (unsigned)items, kChunkThreads, ChunkGeo<D>::kSmem, st, 1,
                                 mq, mk, mv, C, heads, cu_q, kv_len, rows, scale, P.sp.small_rows, P.sp.per[1],
                                 P.sp.splits[1], P.longest ? 1 : 0, ot, out_ld, part + P.sp.part1 * (D + 8), waits))
      return why;
  }
  if (P.decode) {
    const int64_t grid = (int64_t)C.seqs * C.kv_heads * P.sp.splits[0];
    if (grid > 0x7fffffff) return "too many sequences";
    auto* fn = P.join ? k_paged_decode<T, O, D, true> : k_paged_decode<T, O, D, false>;
    const float scale_log2 = std::min(std::max(scale * 1.44269504f, -3.4e38f), 3.4e38f);
    if (!allow_smem(fn, DecodeGeo<D>::kSmem, dev)) return "shared memory could not be set";
    if (const char* why = launch(P.chunk || chained, fn, (unsigned)grid, 32 * kDecodeWarps, DecodeGeo<D>::kSmem, st,
                                 P.join ? P.sp.splits[0] : 1, C, qt, q_ld, heads, cu_q, kv_len, rows, scale_log2,
                                 P.sp.per[0], P.sp.splits[0], P.chunk ? 1 : 0, ot, out_ld, part))
      return why;
  }
  const bool small = P.sp.splits[0] > 1 && !P.join, large = P.sp.splits[1] > 1;  // whose splits are left
  if (small || large) {
    // a group of threads for every kCombineRun splits, as far as a block goes
    const int most = std::max(small ? P.sp.splits[0] : 1, P.sp.splits[1]);
    int groups_log2 = 0;
    while (most > kCombineRun << groups_log2 && D / 8 << groups_log2 < kCombineThreads) ++groups_log2;
    const int tile_rows = (int)std::min<int64_t>(kDecodeRows, (int64_t)std::max(max_q, 1) * (heads / C.kv_heads));
    auto blocks = [&](int64_t units) { return ((units * (D / 8) << groups_log2) + kCombineThreads - 1) / kCombineThreads; };
    const int64_t b0 = small ? blocks((int64_t)C.seqs * C.kv_heads * tile_rows) : 0;
    const int64_t b1 = large ? blocks((int64_t)rows * heads) : 0;
    if (b0 + b1 > 0x7fffffff) return "too many rows";
    if (const char* why = launch(true, k_paged_combine<O, D>, (unsigned)(b0 + b1), kCombineThreads, 0, st, 1, C, heads, cu_q,
                                 kv_len, rows, P.sp, (int)b0, tile_rows, groups_log2, part, ot, out_ld))
      return why;
  }
  return nullptr;
}

// A call of W keys over all its (sequence, kv head) pairs has at most W / (kKeysRoot sqrt(W)) decode
// splits and one more for each pair; chunks make at most kChunkItems (item, split) pairs of two row
// tiles.
size_t attention_bytes_max(int head_dim, int kv_heads, int seqs, int max_kv) {
  const double units = (double)seqs * kv_heads;
  const size_t splits = (size_t)(std::sqrt(units * max_kv) / kKeysRoot + units) + 1;
  return (kDecodeRows * splits + (size_t)2 * kTileRows * kChunkItems) * (head_dim + 8) * sizeof(float);
}

const char* attention_rows(const llama_paged_kv_t* kv, int dev, const void* q, int64_t q_ld, int heads,
                           const int32_t* cu_q, const int32_t* kv_len, int rows, int max_q, int max_kv, float scale,
                           void* out, int out_type, int64_t out_ld, void* workspace, const Waits& waits, cudaStream_t st,
                           bool chained) {
  const Plan P = plan_of(kv, heads, rows, max_q, max_kv);
  const Cache C = cache_of(kv);
  auto run = [&](auto c, auto o) {
    using T = decltype(c);
    using O = decltype(o);
    auto* fn = kv->head_dim == 64 ? attention<T, O, 64> : attention<T, O, 128>;
    return fn(kv, P, C, dev, q, q_ld, heads, cu_q, kv_len, rows, max_q, scale, out, out_ld, static_cast<float*>(workspace), waits,
              st, chained);
  };
  auto by_type = [&](auto c) { return out_type == LLAMA_F32 ? run(c, 0.0f) : run(c, c); };
  return kv->type == LLAMA_F16 ? by_type(__half{}) : by_type(__nv_bfloat16{});
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
  const void* ptrs[] = {kv->v, kv->table, qkv, pos, seq, rope_cos, rope_sin, q_out, kv->slots};
  for (const void* p : ptrs)
    if (dev < 0 || (p && device_of(p) != dev)) return refuse(who, "every pointer must be memory of one CUDA device");
  DeviceGuard dg(dev);
  if (const char* why = append_rows(kv, qkv, type, ld, 1, 0, rows, heads, pos, seq, rope_cos, rope_sin, n_pos, q_out, q_type,
                                    q_ld, static_cast<cudaStream_t>(stream), false))
    return refuse(who, why);
  return 0;
}

LE_API size_t llama_paged_attention_workspace(const llama_paged_kv_t* kv, int heads, int rows, int max_q, int max_kv) {
  using namespace paged;
  if (check_cache(kv) || heads < 1 || heads > 4096 || heads % kv->kv_heads != 0 || rows < 1 || max_q < 0 || max_kv < 0)
    return 0;
  return plan_of(kv, heads, rows, max_q, max_kv).bytes;
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
  if (rows == 0) return 0;
  const Plan P = plan_of(kv, heads, rows, max_q, max_kv);
  if (P.bytes > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < P.bytes))
    return refuse(who, "workspace is too small", -2);
  const int dev = device_of(kv->k);
  const void* ptrs[] = {kv->v, kv->table, q, cu_q, kv_len, out, workspace, kv->slots};
  for (const void* p : ptrs)
    if (dev < 0 || (p && device_of(p) != dev)) return refuse(who, "every pointer must be memory of one CUDA device");
  DeviceGuard dg(dev);
  if (const char* why = attention_rows(kv, dev, q, q_ld, heads, cu_q, kv_len, rows, max_q, max_kv, scale, out, out_type, out_ld,
                                       workspace, Waits(), static_cast<cudaStream_t>(stream), false))
    return refuse(who, why);
  return 0;
}
