// Chunk form of llama_paged_attention: prompt chunks of any length over the paged cache, on the
// tcgen05 tensor cores.
//
//   o = sum_j 2^(c s_j - c m) v_j / sum_j 2^(c s_j - c m),  s_j = q . k_j,  c = scale log2(e)
//
// The G query heads that share a kv head and the n tokens of a sequence form one axis of rows
// (token-major); a row tile is the 128 / G whole tokens that fit the 128 rows of an MMA (G > 128: 128
// of a token's heads), and a work item two row tiles of one sequence and kv head, so that every key is
// read once for up to 256 rows.  One CTA per SM takes items in turn, those with many keys first (a CTA
// that is done takes over the next one of the grid that has not started), and walks an item's keys in
// tiles of 128:
//
//   * warp 9 finds the items and runs ahead of the others: it publishes an item's description and brings Q
//     (one box of heads x tokens per column block).  Warp 9 brings the K rows and warp 10 the V rows,
//     tile by tile into a ring of stages by TMA, one box per page and 64-element column block, straight into the
//     128-byte-swizzled layouts that the MMA reads: K as the K-major operand of S = Q K^T, V (whose
//     rows are keys) as the MN-major operand of O += P V, so nothing is transposed.  Pages past the
//     keys, and page ids out of range, are addressed past the pool's last page: TMA fills them with
//     zeros.  The rows of the last page behind the length may hold anything, NaN too, which a
//     weight of 0 would not silence: the loader zeroes them in the V stage before it hands it over.
//   * warp 8 (one thread) issues the products, alternating between the two row tiles so that one
//     tile's products run while the other's softmax does.  S_i is 128 fp32 columns of tensor memory,
//     P_i 64 columns, O_i head_dim columns.  With head_dim 64 P_i lies beside S_i, and S_i of the
//     next keys is computed as soon as this one has been read; with 128 P_i replaces S_i.  P is handed
//     over in two halves, so that the first half's product runs during the second's exponentials.
//   * warps 0..3 and 4..7 are the softmax of tile 0 and 1, a thread per row (= tensor-memory lane), so
//     that a row's maximum and sum need no exchange.  O is only rescaled when a row's maximum has
//     grown by more than 2^8 since the value it is scaled by; until then weights may exceed 1, by at
//     most 2^8, which costs no accuracy in fp32 sums or 16-bit weights (this and the next are published
//     techniques of tiled attention).  A quarter of the
//     exponentials is computed on the FMA units (range reduction to
//     |f| <= 1/2 and a polynomial of degree 5, 1e-7 relative), since 16 a clock and SM is what the
//     special-function units give.
// Weights are rounded to the cache's type as the A operand of P V; their sum is taken in fp32 before
// that.
//
// All mbarrier waits are bounded; on timeout the engine's error word is set, every role stops, the copies and
// products in flight are waited for (again bounded) and the rows of the items that the CTA had taken on
// become NaN.
//
// Bound by the softmax and its hand-overs: per key tile and row tile the products take 1,030 clocks
// (head_dim 128; 770 with 64, whose MN-major V of 64 columns runs at half rate), the softmax's 128 x 128
// exponentials 770 on the special-function units and about 1,150 with the maxima, sums, conversions and
// tensor-memory reads around them; two row tiles are under way at a time, and a key tile of both takes
// 3,300 clocks with heads of 128.  One sequence of 8192 tokens, 32 heads: head_dim
// 128 458 us (1201 TFLOP/s), 64 401 us (685).  512 tokens over 32768 keys, heads of 128: 251 us (1085) in a
// burst, 283 to 295 us in a row of calls, under the power cap.  8 x 2048, heads of 64: 250 us (550), 3,900
// clocks for a key tile of both row tiles, of which the arithmetic above explains 2,300: an item has 8.5 key
// tiles here, its softmax warps themselves wait for its last product, read O and store it, and the diagonal
// key tiles are computed whole.  Tried and no faster: 16 softmax warps, one pass over S held
// in registers, a product warp for each row tile, other shares of polynomial exponentials (0, 3/8, 1/2).
#pragma once

#include <cuda.h>

#include "ops.h"
#include "paged.cuh"
#include "ptx.cuh"

namespace le {
namespace paged {

constexpr int kTileRows = 128;                 // rows of an MMA tile
constexpr int kTileKeys = 128;
constexpr int kChunkThreads = 352;             // 2 x 4 softmax warps, products, two loaders
constexpr int kBlockBytes = kTileKeys * 128;   // one 64-element column block of 128 rows
constexpr float kLazyLog2 = 8.0f;              // growth of a maximum that forces a rescale (log2)
template <int D> struct ChunkGeo {
  static constexpr int kCols = D / 64;                       // column blocks of a row
  static constexpr int kStageBytes = kCols * kBlockBytes;    // K or V of a key tile, or Q of a row tile
  static constexpr int kStages = D == 64 ? 8 : 5;
  static constexpr int kQBufs = D == 64 ? 2 : 1;             // items whose Q is held
  static constexpr int kSmem = 1024 + (2 * kQBufs + kStages) * kStageBytes;
  // tensor memory (all 512 columns): S_i, P_i and O_i of the two row tiles
  static constexpr bool kApart = D == 64;                    // P beside S
  static constexpr uint32_t kColP = kApart ? 256 : 0, kStepP = kApart ? 64 : 128, kColO = 512 - 2 * D;
};

// Descriptor of a 128-byte-swizzled operand whose 16-bit elements run along N (MN-major): 64-element
// column blocks kBlockBytes apart (leading byte offset), 8-key groups 1024 bytes apart.
__device__ __forceinline__ uint64_t mn_desc(uint32_t saddr) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(kBlockBytes >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// Instruction descriptor, kind::f16, fp32 accumulator, M = 128: element format in A and B, B along
// K (0) or along N (1).
template <typename T>
__device__ __forceinline__ constexpr uint32_t chunk_idesc(int n, int b_mn) {
  constexpr uint32_t f = std::is_same<T, __half>::value ? 0u : 1u;
  return (1u << 4) | (f << 7) | (f << 10) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void chunk_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, int x, int head, int row, int page,
                                        uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
          dst),
      "l"(map), "r"(bar), "r"(x), "r"(head), "r"(row), "r"(page)
      : "memory");
}
__device__ __forceinline__ void tma_rows(uint32_t dst, const CUtensorMap* map, int x, int head, int row, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          dst),
      "l"(map), "r"(bar), "r"(x), "r"(head), "r"(row)
      : "memory");
}
template <int N>
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* v) {
  static_assert(N == 16, "16 columns");
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

constexpr uint32_t kNegInf = 0xff800000u;
// Largest of three; NaN if one is.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 w, x, y;\n\t"
      "mov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// Waits (bounded) for phase `parity`; false after a timeout here or elsewhere in the CTA.  Every lane that
// goes on to read what the phase guards polls for itself: what other threads and the asynchronous copies wrote
// before it (an item, the answer of a takeover) is visible to those that saw it complete.  A lane that
// polled for its warp and passed the outcome on by a shuffle, which orders no memory, would leave the others
// with old items to make addresses from.
__device__ __forceinline__ bool chunk_wait(uint32_t bar, uint32_t parity, volatile uint32_t* abort, const Waits& W) {
  unsigned long long t0 = 0;
  for (uint32_t n = 1;; ++n) {
    if (mbar_try(bar, parity)) return true;
    if ((n & 15u) == 0) {  // now and then: has another thread given up, or the time run out?
      if (*abort) return false;
      const unsigned long long t = gtimer();
      if (t0 == 0) t0 = t;
      if (t - t0 > W.ns) {
        *abort = 1u;
        return false;
      }
    }
  }
}
__device__ __forceinline__ void chunk_drain(uint32_t bar, uint32_t parity, const Waits& W) {
  const unsigned long long t0 = gtimer();
  while (!mbar_try(bar, parity) && gtimer() - t0 < W.ns) {
  }
}

// 2^x for a pair: x = n + f, n the nearest integer, 2^f by a polynomial of degree 5 fitted to the
// smallest relative error on |f| <= 1/2 (9e-8), n added to the exponent.  x below -126 counts as -126.
__device__ __forceinline__ float2 exp2_poly(float2 x) {
  constexpr float kMagic = 12582912.0f;  // 1.5 2^23: adding it rounds to an integer
  x.x = fmaxf(x.x, -126.0f);
  x.y = fmaxf(x.y, -126.0f);
  const float2 t = add2(x, make_float2(kMagic, kMagic));
  const float2 n = add2(t, make_float2(-kMagic, -kMagic));
  const float2 f = fma2(n, make_float2(-1.0f, -1.0f), x);
  float2 p = fma2(make_float2(1.32647292e-3f, 1.32647292e-3f), f, make_float2(9.67151344e-3f, 9.67151344e-3f));
  p = fma2(p, f, make_float2(5.55073375e-2f, 5.55073375e-2f));
  p = fma2(p, f, make_float2(2.40222421e-1f, 2.40222421e-1f));
  p = fma2(p, f, make_float2(6.93146978e-1f, 6.93146978e-1f));
  p = fma2(p, f, make_float2(1.0f, 1.0f));
  return make_float2(__uint_as_float(__float_as_uint(p.x) + (__float_as_uint(t.x) << 23)),
                     __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(t.y) << 23)));
}

// Takes over a CTA of this grid that has not started (16 bytes to shared memory, on a barrier): the SM
// that is done first gets the next item, without a counter in memory.
__device__ __forceinline__ void steal_cta(uint32_t to, uint32_t bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(to),
               "r"(bar)
               : "memory");
}
// Its block index, or -1 when every CTA has started.
__device__ __forceinline__ int stolen_cta(uint32_t from) {
  uint32_t got, x;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 r;\n\tld.shared.b128 r, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\tselp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n\t}"
      : "=r"(got), "=r"(x)
      : "r"(from)
      : "memory");
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // read before the next one is written
  return got ? (int)x : -1;
}

// How rows are cut into tiles: `tokens` tokens of `heads` heads a tile, `parts` tiles across a token's
// heads (more than one only for G > 128).
struct RowTiles {
  int G, heads, tokens, parts;
};
__host__ __device__ __forceinline__ RowTiles row_tiles(int G) {
  RowTiles t;
  t.G = G;
  t.heads = G < kTileRows ? G : kTileRows;
  t.tokens = kTileRows / t.heads;
  t.parts = (G + kTileRows - 1) / kTileRows;
  return t;
}

// A work item as its CTA's roles see it.
struct Item {
  int seq;           // -1: no more
  int g, z, used;    // kv head, key split, splits of the sequence
  int first, n, len; // rows and keys of the sequence
  int unit;          // first of the item's two row tiles
  int k_lo;          // first key of the split
  int nk[2];         // key tiles that the row tiles see
};
// Items of a sequence (two row tiles each), and those of them that see more than `keys` keys (all of them
// for keys < 0): item j's last token is the ((2 j + 1) / parts + 1) tokens-th, so they are the last ones.
__device__ __forceinline__ int items_of(const Span& sp, const RowTiles& T, int small_rows) {
  return sp.n <= 0 || sp.n * T.G <= small_rows ? 0 : ((sp.n + T.tokens - 1) / T.tokens * T.parts + 1) / 2;
}
__device__ __forceinline__ int items_above(const Span& sp, const RowTiles& T, int items, int keys) {
  const int y = keys - (sp.len - sp.n);
  return keys < 0 || y < 0 ? items : y >= sp.n ? 0 : items - min(items, T.parts * (y / T.tokens) / 2);
}
// Item w of the launch: kv heads fastest, then splits, then the pairs of row tiles.  longest (at most 32
// sequences): the pairs in order of the key tiles they see, the most first, so that the last items are
// short ones; otherwise the sequences from the last to the first, each from its last pair to its first,
// which keeps a sequence's keys in L2 while they are used.  Found by
// a whole warp; the result is the same in every lane.
__device__ __forceinline__ Item find_item(const Cache& C, const int32_t* cu_q, const int32_t* kv_len, int rows,
                                          const RowTiles& T, int small_rows, int per, int splits, int total, int longest,
                                          int w) {
  const int lane = threadIdx.x & 31;
  Item it;
  it.seq = -1;
  if (w < 0) return it;
  it.g = w % C.kv_heads;
  it.z = (w / C.kv_heads) % splits;
  int want = w / C.kv_heads / splits;
  if (want >= total) return it;
  int before = 0, local = 0;
  if (longest) {
    Span sp{0, 0, 0};
    if (lane < C.seqs) sp = span_of(C, cu_q, kv_len, lane, rows);
    const int items = items_of(sp, T, small_rows);
    auto above = [&](int tiles) { return items_above(sp, T, items, tiles * kTileKeys); };
    // the item sees more than lo key tiles and at most hi
    int lo = -1, hi = ((int)__reduce_max_sync(0xffffffffu, (unsigned)sp.len) + kTileKeys - 1) / kTileKeys;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if ((int)__reduce_add_sync(0xffffffffu, (unsigned)above(mid)) > want) lo = mid;
      else hi = mid;
    }
    const int longer = above(hi), here = above(lo);
    want -= (int)__reduce_add_sync(0xffffffffu, (unsigned)longer);
    int inc = here - longer;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    it.seq = __ffs(__ballot_sync(0xffffffffu, inc > want)) - 1;
    local = __shfl_sync(0xffffffffu, items - here + want - (inc - (here - longer)), max(it.seq, 0));
  } else {
    want = total - 1 - want;
    for (int s0 = 0; s0 < C.seqs && it.seq < 0; s0 += 32) {
      const int mine = s0 + lane < C.seqs ? items_of(span_of(C, cu_q, kv_len, s0 + lane, rows), T, small_rows) : 0;
      int inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + inc > want);
      if (hit) {
        const int l = __ffs(hit) - 1;
        it.seq = s0 + l;
        local = want - before - __shfl_sync(0xffffffffu, inc - mine, l);
      }
      before += __shfl_sync(0xffffffffu, inc, 31);
    }
  }
  if (it.seq < 0) return it;
  const Span sp = span_of(C, cu_q, kv_len, it.seq, rows);
  it.first = sp.first;
  it.n = sp.n;
  it.len = sp.len;
  it.unit = 2 * local;
  it.used = splits_of(sp.len, per, splits);
  it.k_lo = it.z * per;
  const int units = (sp.n + T.tokens - 1) / T.tokens * T.parts;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    // keys of the tile's rows: all up to its last row's position, within this split
    const int last = min((it.unit + i) / T.parts * T.tokens + T.tokens, sp.n) - 1;
    int end = it.unit + i < units && it.z < it.used ? min(sp.len, sp.len - sp.n + last + 1) : 0;
    if (it.z != splits - 1) end = min(end, it.k_lo + per);
    it.nk[i] = end > it.k_lo ? (end - it.k_lo + kTileKeys - 1) / kTileKeys : 0;
  }
  return it;
}
// Row tiles of the whole call, two an item.
__device__ __forceinline__ int count_items(const Cache& C, const int32_t* cu_q, const int32_t* kv_len, int rows,
                                           const RowTiles& T, int small_rows) {
  const int lane = threadIdx.x & 31;
  int total = 0;
  for (int s = lane; s < C.seqs; s += 32) total += items_of(span_of(C, cu_q, kv_len, s, rows), T, small_rows);
  return (int)__reduce_add_sync(0xffffffffu, (unsigned)total);
}

// A softmax thread's row of an item.
struct Row {
  int tok, h;      // row of q and out, query head
  int lim;         // last key it sees
  int lim_first;   // the tile's first row's
  bool live;       // exists
};
__device__ __forceinline__ Row row_of(const Item& it, const RowTiles& T, int i, int r) {
  Row x;
  const int unit = it.unit + i, t0 = unit / T.parts * T.tokens, head = unit % T.parts * kTileRows + r % T.heads;
  const int tok = t0 + r / T.heads, last = min(t0 + T.tokens, it.n) - 1;
  x.live = r < T.tokens * T.heads && tok < it.n && head < T.G;
  x.tok = it.first + min(tok, it.n - 1);
  x.h = it.g * T.G + min(head, T.G - 1);
  x.lim_first = it.len - it.n + t0;
  x.lim = it.len - it.n + min(tok, last);  // rows that do not exist see what the last one does
  return x;
}

// Grid: at least one CTA for every item x split x kv head (find_item's order).  per: keys of a split, a multiple of 128.
// Sequences of at most small_rows rows per kv head are the decode form's.
template <typename T, typename O, int D>
__global__ void __launch_bounds__(kChunkThreads, 1)
    k_paged_chunk(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, Cache C, int heads, const int32_t* __restrict__ cu_q,
                  const int32_t* __restrict__ kv_len, int rows, float scale, int small_rows, int per, int splits, int longest,
                  O* __restrict__ out, int64_t out_ld, float* __restrict__ part, Waits W) {
  using Geo = ChunkGeo<D>;
  constexpr int kSt = Geo::kStages, kQb = Geo::kQBufs;
  extern __shared__ uint8_t chunk_smem[];
  // barriers: stage full, stage empty; item published, item read; Q full, Q empty; then per row tile S
  // ready, S read, P halves, O done, O read; the loader's own for a V tail; one that nothing completes
  constexpr int kFull = 0, kEmpty = kSt, kItem = 2 * kSt, kItemFree = kItem + 2, kQFull = kItemFree + 2, kQEmpty = kQFull + kQb;
  constexpr int kBarS = kQEmpty + kQb, kBarR = kBarS + 2, kBarP = kBarR + 2, kBarO = kBarP + 4, kBarE = kBarO + 2;
  constexpr int kBarFix = kBarE + 2, kNever = kBarFix + 1, kSteal = kNever + 1, kBars = kSteal + 1;
  __shared__ __align__(8) unsigned long long s_bar[kBars];
  __shared__ Item s_item[2];
  __shared__ __align__(16) uint32_t s_steal[4];
  __shared__ volatile int s_claimed[4], s_claims;  // the launch's items that this CTA has taken on: the last four, how many
  __shared__ uint32_t s_tmem;
  __shared__ volatile uint32_t s_abort;
  __shared__ volatile uint32_t s_live[16];  // per key tile: bit x, its keys 16 x .. 16 x + 15 have a page
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  auto bar = [&](int i) { return smem_u32(&s_bar[i]); };
  if (tid == 0) {
    s_abort = 0u;
    s_claims = 0;
    for (int i = 0; i < kBars; ++i) {
      const bool half = (i >= kBarR && i < kBarO) || (i >= kBarE && i < kBarFix);       // a row tile's threads
      mbar_init(bar(i), half ? kTileRows : i == kItemFree || i == kItemFree + 1 ? 10 : 1);  // the item's readers
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) {
    tc::tmem_alloc(smem_u32(&s_tmem), 512);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  grid_dep_wait();
  grid_dep_launch();  // the decode form of the same call may start: its inputs are complete
  const uint32_t tmem = s_tmem;
  const RowTiles R = row_tiles(heads / C.kv_heads);
  const uint32_t base = (smem_u32(chunk_smem) + 1023u) & ~1023u;  // Q buffers of two row tiles, then the stages
  const uint32_t stage0 = base + (uint32_t)(2 * kQb * Geo::kStageBytes);
  const int page_mask = (1 << C.page_log2) - 1;
  int item = 1 << 30;  // the item that a wait which ran out ended
  if (warp >= 8) {
    if (warp >= 9) {
      // ---- loaders: K (and the items and Q), V ----
      const int kv = warp - 9;
      const int total = kv == 0 ? count_items(C, cu_q, kv_len, rows, R, small_rows) : 0;
      const int box = min(1 << C.page_log2, kTileKeys), boxes = kTileKeys / box;
      const CUtensorMap* const map = kv ? &map_v : &map_k;
      const bool leader = tc::elect_one();
      bool ok = true;
      int fills = 0, tiles = 0, fixes = 0, qs = 0, last = -1;  // fills: K and V of a tile are two
      auto wait = [&](int b, int n) { return __all_sync(0xffffffffu, chunk_wait(bar(b), (uint32_t)n & 1u, &s_abort, W)); };
      int w = blockIdx.x, steals = 0;
      auto steal = [&] {
        if (leader) {
          mbar_expect_tx(bar(kSteal), 16);
          steal_cta(smem_u32(s_steal), bar(kSteal));
        }
        ++steals;
      };
      auto stolen = [&] {  // the next item; -1: no more, or a wait ran out
        ok = wait(kSteal, steals - 1);
        w = ok ? __shfl_sync(0xffffffffu, stolen_cta(smem_u32(s_steal)), 0) : -1;  // the warp's, as find_item wants it
        __syncwarp();
      };
      for (int k = 0; ok; ++k) {
        Item it;
        if (kv == 0) {
          do {  // past the last item the launch has CTAs without work
            it = find_item(C, cu_q, kv_len, rows, R, small_rows, per, splits, total, longest, w);
            if (it.seq < 0 && w >= 0) {
              steal();
              stolen();
            }
          } while (ok && it.seq < 0 && w >= 0);
          if (it.seq >= 0) {
            if (leader) {
              s_claimed[k & 3] = w;
              s_claims = k + 1;
            }
            steal();  // the answer is there when this item has been loaded
          }
          if (ok && k >= 2) ok = wait(kItemFree + (k & 1), k / 2 - 1);
          if (!ok) break;
          if (leader) {
            s_item[k & 1] = it;
            mbar_arrive_n(bar(kItem + (k & 1)), 1);
          }
        } else {
          ok = wait(kItem + (k & 1), k / 2);
          if (!ok) break;
          it = s_item[k & 1];
          __syncwarp();
          if (leader) mbar_arrive_n(bar(kItemFree + (k & 1)), 1);
        }
        if (it.seq < 0) break;
        const int nk = max(it.nk[0], it.nk[1]);
        if (nk == 0) {
          if (kv == 0) stolen();
          continue;
        }
        if (kv == 0) {
          if (qs >= kQb) ok = wait(kQEmpty + qs % kQb, qs / kQb - 1);
          if (!ok) break;
          const int b = qs % kQb, tile_bytes = R.tokens * R.heads * 128 * Geo::kCols;
          const int both = it.nk[1] > 0 ? 2 : 1;
          if (leader) {
            mbar_expect_tx(bar(kQFull + b), (uint32_t)(both * tile_bytes));
            for (int i = 0; i < both; ++i)
#pragma unroll
              for (int cb = 0; cb < Geo::kCols; ++cb)
                tma_rows(base + (uint32_t)((2 * b + i) * Geo::kStageBytes + cb * kBlockBytes), &map_q, cb * 64,
                         it.g * R.G + (it.unit + i) % R.parts * kTileRows, it.first + (it.unit + i) / R.parts * R.tokens,
                         bar(kQFull + b));
          }
          __syncwarp();
          ++qs;
        }
        // the key tile that reaches past the length inside a page (the item's last one), if any
        const int fix = kv && (it.len & page_mask) != 0 && it.k_lo + nk * kTileKeys > it.len ? nk - 1 : -1;
        const int32_t* table = pages_of(C, it.seq);
        const int k_hi = min(it.len, it.k_lo + nk * kTileKeys);  // keys that are loaded
        // this lane's page of tile j as the table has it, loaded a tile ahead and looked at only then;
        // 0 where no key is wanted
        auto entry_of = [&](int j) {
          const int key = it.k_lo + j * kTileKeys + lane * box, e = key >> C.page_log2;
          return table && lane < boxes && key < k_hi && e < C.table_width ? table[e] : 0;
        };
        int entry = entry_of(0);
        for (int j = 0; j < nk && ok; ++j, ++tiles) {
          const int next = j + 1 < nk ? entry_of(j + 1) : 0;
          const int row = (it.k_lo + j * kTileKeys) & page_mask;  // nonzero only where pages exceed a tile
          const bool wanted = lane < boxes && it.k_lo + j * kTileKeys + lane * box < k_hi;
          const bool valid = table && entry >= 0 && entry < C.num_pages;
          const int page = wanted && valid ? entry : C.num_pages;  // none: behind the pool's last
          const int f = fills + 2 * j + kv, st = f % kSt;
          if (f >= kSt) ok = wait(kEmpty + st, f / kSt - 1);
          if (!ok) break;
          if (kv == 0) {
            const unsigned gone = __ballot_sync(0xffffffffu, wanted && !valid);
            uint32_t live = 0xffu;
            for (int x = 0; gone && x < 8; ++x)
              if ((gone >> (16 * x / box)) & 1u) live &= ~(1u << x);
            if (leader) s_live[tiles & 15] = live;
          }
          // a stage whose tail is zeroed lands on a barrier of the loader's own first
          const uint32_t landed = bar(j == fix ? kBarFix : kFull + st);
          const uint32_t to = stage0 + (uint32_t)(st * Geo::kStageBytes);
          if (leader) mbar_expect_tx(landed, Geo::kStageBytes);
          __syncwarp();
          last = f;
          // one lane issues the boxes, one after the other: their operands are the warp's
          auto issue = [&](auto count) {
            constexpr int n = decltype(count)::value;
            int pg[n];
#pragma unroll
            for (int x = 0; x < n; ++x) pg[x] = __shfl_sync(0xffffffffu, page, x);
            if (leader) {
#pragma unroll
              for (int x = 0; x < n; ++x)
#pragma unroll
                for (int cb = 0; cb < Geo::kCols; ++cb)
                  tma_box(to + (uint32_t)(cb * kBlockBytes + x * (kTileKeys / n) * 128), map, cb * 64, it.g, row, pg[x], landed);
            }
          };
          if (boxes == 8) issue(std::integral_constant<int, 8>{});
          else if (boxes == 4) issue(std::integral_constant<int, 4>{});
          else if (boxes == 2) issue(std::integral_constant<int, 2>{});
          else issue(std::integral_constant<int, 1>{});
          if (j == fix) {
            ok = wait(kBarFix, fixes++);
            const int r0 = it.len - (it.k_lo + j * kTileKeys);  // first row behind the length
            for (int i = lane; i < (kTileKeys - r0) * 8 * Geo::kCols; i += 32) {
              const int cb = i / ((kTileKeys - r0) * 8), x = i % ((kTileKeys - r0) * 8);
              const uint32_t a = to + (uint32_t)(cb * kBlockBytes + r0 * 128 + x * 16);
              asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(a), "r"(0u) : "memory");
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (leader && ok) mbar_arrive_n(bar(kFull + st), 1);
          }
          entry = next;
        }
        fills += 2 * nk;
        if (kv == 0 && ok) stolen();
      }
      if (s_abort) {  // the copies in flight land before the shared memory goes
        for (int f = last; f >= 0 && f > last - kSt; f -= 2) chunk_drain(bar(kFull + f % kSt), (uint32_t)(f / kSt) & 1u, W);
        for (int f = max(0, qs - kQb); f < qs; ++f) chunk_drain(bar(kQFull + f % kQb), (uint32_t)(f / kQb) & 1u, W);
        if (fixes > 0) chunk_drain(bar(kBarFix), (uint32_t)(fixes - 1) & 1u, W);
        if (steals > 0) {  // an item that was taken on but not begun is among those that become NaN
          chunk_drain(bar(kSteal), (uint32_t)(steals - 1) & 1u, W);
          const int next = w >= 0 || !ok ? stolen_cta(smem_u32(s_steal)) : -1;
          const int n = s_claims;
          __syncwarp();
          if (leader && next >= 0 && (n == 0 || s_claimed[(n - 1) & 3] != next)) {
            s_claimed[n & 3] = next;
            s_claims = n + 1;
          }
        }
      }
    } else if (warp == 8) {
      // ---- products ----
      constexpr uint32_t id_o = chunk_idesc<T>(D, 1);
      const uint32_t id_s = chunk_idesc<T>(kTileKeys, 0) | (scale < 0.0f ? 1u << 13 : 0u);  // A = -Q: |scale| remains
      // What the products' operands are made of has to be the warp's in the compiler's eyes as well (a
      // reduction's result is): else every operand goes through a register of one lane.
      const uint32_t t0 = __reduce_max_sync(0xffffffffu, tmem);
      const bool leader = tc::elect_one();
      bool ok = true;
      int st = 0, ph = 0;  // stage and phase of the next fill (K and V of a tile are two)
      int q = 0, qp = 0;   // Q buffer and phase of the next item
      int tiles[2] = {0, 0}, reads[2] = {0, 0};  // per row tile: key tiles so far, items that had some
      int last = -1, last_parity = 0;
      auto wait = [&](int b, int n) { return __all_sync(0xffffffffu, chunk_wait(bar(b), (uint32_t)n & 1u, &s_abort, W)); };
      auto commit = [&](int b, int n) {  // n: the phase that this completes
        if (leader) tc::tc_commit(bar(b));
        last = b;
        last_parity = n & 1;
      };
      if (W.expire) ok = wait(kNever, 0);  // test only
      for (int k = 0; ok; ++k) {
        ok = wait(kItem + (k & 1), k / 2);
        if (!ok) break;
        const bool more = __reduce_max_sync(0xffffffffu, s_item[k & 1].seq) >= 0;
        const int nk0 = __reduce_max_sync(0xffffffffu, s_item[k & 1].nk[0]), nk1 = __reduce_max_sync(0xffffffffu, s_item[k & 1].nk[1]);
        if (lane == 0) mbar_arrive_n(bar(kItemFree + (k & 1)), 1);
        if (!more) break;
        const int nk = max(nk0, nk1);
        if (nk == 0) continue;
        // S_i from the K in stage s
        auto issue_s = [&](int i, int j, int s) {
          const uint32_t a = base + (uint32_t)((2 * q + i) * Geo::kStageBytes), b = stage0 + (uint32_t)(s * Geo::kStageBytes);
          tc::tc_fence_after();
          if (leader) {
#pragma unroll
            for (int x = 0; x < D / 16; ++x) {
              const uint32_t off = (uint32_t)((x >> 2) * kBlockBytes);
              chunk_mma_ss(t0 + 128u * i, tc::sw128_desc(a + off) + 2 * (x & 3), tc::sw128_desc(b + off) + 2 * (x & 3), id_s,
                           x > 0 ? 1u : 0u);
            }
          }
          commit(kBarS + i, tiles[i] + j);
        };
        ok = wait(kQFull + q, qp) && wait(kFull + st, ph);
        if (!ok) break;
        if (Geo::kApart && nk0 > 0 && tiles[0] > 0) ok = wait(kBarR + 0, tiles[0] - 1);
        if (ok && nk0 > 0) issue_s(0, 0, st);
        if (ok && Geo::kApart && nk1 > 0 && tiles[1] > 0) ok = wait(kBarR + 1, tiles[1] - 1);
        if (ok && nk1 > 0) issue_s(1, 0, st);
        if (!ok) break;
        commit(kEmpty + st, ph);
        if (nk == 1) commit(kQEmpty + q, qp);
        if (++st == kSt) st = 0, ++ph;
        for (int j = 0; j < nk && ok; ++j) {
          const int sv = st, pv = ph;
          if (++st == kSt) st = 0, ++ph;
          const int sk = st, pk = ph;  // K of the next tile
          const bool next = j + 1 < nk;
          if (next && ++st == kSt) st = 0, ++ph;
          const uint32_t v = stage0 + (uint32_t)(sv * Geo::kStageBytes);
          ok = wait(kFull + sv, pv) && (!next || wait(kFull + sk, pk));
          // the order in which the softmax warps get to them: P_i V and S_i of the next keys (with P apart
          // as soon as this one's columns have been read; in place behind the product that reads P_i)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int nki = i ? nk1 : nk0;
            if (!ok || j >= nki) continue;
            if (Geo::kApart && j + 1 < nki) {
              ok = wait(kBarR + i, tiles[i] + j);
              if (!ok) continue;
              issue_s(i, j + 1, sk);
            }
            if (j == 0 && reads[i] > 0) ok = wait(kBarE + i, reads[i] - 1);  // O_i of the item before has been read
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              ok = ok && wait(kBarP + 2 * i + half, tiles[i] + j);
              if (!ok) break;
              tc::tc_fence_after();
              if (leader) {
#pragma unroll
                for (int x = 4 * half; x < 4 * half + 4; ++x)  // 16 keys: 8 columns of P, 2048 bytes of V
                  tc::tc_mma_ts(t0 + Geo::kColO + (uint32_t)(D * i), t0 + Geo::kColP + Geo::kStepP * i + 8u * x,
                                mn_desc(v + 2048u * x), id_o, (j > 0 || x > 0) ? 1u : 0u);
              }
            }
            if (!ok) continue;
            commit(kBarO + i, tiles[i] + j);
            if (!Geo::kApart && j + 1 < nki) issue_s(i, j + 1, sk);
          }
          if (!ok) break;
          commit(kEmpty + sv, pv);
          if (next) commit(kEmpty + sk, pk);
          if (j + 2 == nk) commit(kQEmpty + q, qp);
        }
        if (!ok) break;
        tiles[0] += nk0;
        tiles[1] += nk1;
        reads[0] += nk0 > 0 ? 1 : 0;
        reads[1] += nk1 > 0 ? 1 : 0;
        if (++q == kQb) q = 0, ++qp;
      }
      // the last commit covers every product before it: none outlives the tensor and shared memory
      if (last >= 0) chunk_drain(bar(last), (uint32_t)last_parity, W);
      __syncwarp();
    }
  } else {
    // ---- softmax of row tile i, a thread per row ----
    const int i = warp >> 2;
    // > 0, since a masked -inf has to stay -inf, but too small for any score where the scale is 0; and finite
    const float c = fminf(fmaxf(fabsf(scale) * 1.44269504f, 1e-45f), 3.4e38f);
    const uint32_t lanes = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
    const uint32_t t_s = lanes + 128u * i, t_p = lanes + Geo::kColP + Geo::kStepP * i, t_o = lanes + Geo::kColO + (uint32_t)(D * i);
    bool ok = true;
    int tiles = 0, all_tiles = 0, k = 0;
    auto wait = [&](int b, int n) { return __all_sync(0xffffffffu, chunk_wait(bar(b), (uint32_t)n & 1u, &s_abort, W)); };
    for (;; ++k) {
      ok = wait(kItem + (k & 1), k / 2);
      if (!ok) break;
      const Item it = s_item[k & 1];
      __syncwarp();
      if (lane == 0) mbar_arrive_n(bar(kItemFree + (k & 1)), 1);
      if (it.seq < 0) break;
      const Row row = row_of(it, R, i, tid & 127);
      const int nk = i ? it.nk[1] : it.nk[0];
      float m = -INFINITY, l = 0.0f;  // the maximum that O and l are scaled by, and the sum
      for (int j = 0; j < nk; ++j, ++tiles) {
        ok = wait(kBarS + i, tiles);
        if (!ok) break;
        tc::tc_fence_after();
        const int rel = row.lim - (it.k_lo + j * kTileKeys);  // keys 0 .. rel of the tile are seen
        const uint32_t live = s_live[(all_tiles + j) & 15];
        const bool masked = it.k_lo + j * kTileKeys + kTileKeys - 1 > row.lim_first || live != 0xffu;
        // two passes over S, half a tile at a time (the loops are not unrolled: with the code of all 128
        // keys in a row the other warps' instructions no longer stay in the cache)
        float mt = -INFINITY;
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          uint32_t u[2][32];
          tc::tmem_ld32(t_s + 64u * half, u[0]);
          tc::tmem_ld32(t_s + 64u * half + 32u, u[1]);
          tc::tmem_wait_ld();
          if (masked) {
            const int r = rel - 64 * half;
            const uint32_t lv = live >> (4 * half);
#pragma unroll
            for (int x = 0; x < 64; ++x) u[x >> 5][x & 31] = x <= r && ((lv >> (x / 16)) & 1u) ? u[x >> 5][x & 31] : kNegInf;
          }
          float mx[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const uint32_t* v = &u[x >> 1][16 * (x & 1)];
            mx[x] = max3(__uint_as_float(v[0]), __uint_as_float(v[1]), __uint_as_float(v[2]));
#pragma unroll
            for (int e = 3; e < 15; e += 2) mx[x] = max3(mx[x], __uint_as_float(v[e]), __uint_as_float(v[e + 1]));
          }
          mx[0] = max3(mx[0], __uint_as_float(u[0][15]), __uint_as_float(u[0][31]));
          mx[1] = max3(mx[1], __uint_as_float(u[1][15]), __uint_as_float(u[1][31]));
          mt = max3(mt, max3(mx[0], mx[1], mx[2]), mx[3]);
        }
        l = mt == mt ? l : mt;  // a score is NaN, so the row is: not all of the exponentials would pass it on
        // the product of the tile before: with P apart it may still read P and write O (in place, S was
        // computed behind it)
        if (Geo::kApart && tiles > 0) {
          ok = wait(kBarO + i, tiles - 1);
          if (!ok) break;
          tc::tc_fence_after();
        }
        const bool grow = j == 0 ? mt > m : (mt - m) * c > kLazyLog2;
        if (__any_sync(0xffffffffu, grow)) {
          const float alpha = grow ? exp2_approx((m - mt) * c) : 1.0f;
          m = grow ? mt : m;
          l *= alpha;
          if (j > 0) {
#pragma unroll 1
            for (int x = 0; x < D / 16; ++x) {
              uint32_t v[16];
              tc::tmem_ld16(t_o + 16u * x, v);
              tc::tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * alpha);
              tmem_st16<16>(t_o + 16u * x, v);
            }
          }
        }
        const float mc = m == -INFINITY ? 0.0f : m * c;
        const float2 c2 = make_float2(c, c), mc2 = make_float2(-mc, -mc);
        float2 sum0 = make_float2(0.0f, 0.0f), sum1 = make_float2(0.0f, 0.0f);
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          uint32_t u[2][32];
          tc::tmem_ld32(t_s + 64u * half, u[0]);
          tc::tmem_ld32(t_s + 64u * half + 32u, u[1]);
          tc::tmem_wait_ld();
          if (Geo::kApart && half) {  // S may be overwritten
            tc::tc_fence_before();
            mbar_arrive_n(bar(kBarR + i), 1);
          }
          float2 y[2][16];
#pragma unroll
          for (int x = 0; x < 32; ++x) {
            float2& w = y[x >> 4][x & 15];
            w = fma2(make_float2(__uint_as_float(u[x >> 4][2 * (x & 15)]), __uint_as_float(u[x >> 4][2 * (x & 15) + 1])), c2, mc2);
            if (x % 4 == 1) {
              w = exp2_poly(w);
            } else {
              w.x = exp2_approx(w.x);
              w.y = exp2_approx(w.y);
            }
          }
          if (masked) {  // weights of keys that are not seen are exactly 0
            const int r = rel - 64 * half;
            const uint32_t lv = live >> (4 * half);
#pragma unroll
            for (int x = 0; x < 32; ++x) {
              float2& w = y[x >> 4][x & 15];
              const bool lx = (lv >> (x / 8)) & 1u;
              w.x = 2 * x <= r && lx ? w.x : 0.0f;
              w.y = 2 * x + 1 <= r && lx ? w.y : 0.0f;
            }
          }
          uint32_t p[2][16];
#pragma unroll
          for (int x = 0; x < 32; ++x) {
            const float2 w = y[x >> 4][x & 15];
            if (x & 1) sum1 = add2(sum1, w);
            else sum0 = add2(sum0, w);
            p[x >> 4][x & 15] = pack2<T>(w.x, w.y);
          }
          tmem_st16<16>(t_p + 32u * half, p[0]);
          tmem_st16<16>(t_p + 32u * half + 16u, p[1]);
          tc::tmem_wait_st();
          tc::tc_fence_before();
          mbar_arrive_n(bar(kBarP + 2 * i + half), 1);
        }
        l += (sum0.x + sum0.y) + (sum1.x + sum1.y);
      }
      if (ok && nk > 0) {
        ok = wait(kBarO + i, tiles - 1);
        tc::tc_fence_after();
      }
      if (!ok) break;
      // ---- result: the row's D outputs, or this split's part of them ----
      const float inv = l > 0.0f ? 1.0f / l : l == l ? 0.0f : l;  // no key: zeros
      const bool whole = it.used == 1, write = row.live && it.z < it.used;
      float* pp = part + (((int64_t)row.tok * heads + row.h) * splits + it.z) * (D + 8);
      O* po = out + (int64_t)row.tok * out_ld + (int64_t)row.h * D;
#pragma unroll
      for (int x = 0; x < D / 32; ++x) {
        uint32_t v[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = 0u;
        if (nk > 0) {
          tc::tmem_ld32(t_o + 32u * x, v);
          tc::tmem_wait_ld();
        }
        if (write) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            float a[8];
#pragma unroll
            for (int y = 0; y < 8; ++y) a[y] = __uint_as_float(v[e + y]) * (whole ? inv : 1.0f);
            if (whole) store8(po + 32 * x + e, a);
            else store8(pp + 32 * x + e, a);
          }
        }
      }
      if (write && !whole) *reinterpret_cast<float2*>(pp + D) = make_float2(m == -INFINITY ? m : m * c, l);
      if (nk > 0) {
        tc::tc_fence_before();
        mbar_arrive_n(bar(kBarE + i), 1);
      }
      all_tiles += max(it.nk[0], it.nk[1]);
    }
    item = ok ? 1 << 30 : k;
  }
  tc::tc_fence_before();
  __syncthreads();
  // a wait ran out: the rows of the item it ended, and of those that this CTA had taken on behind it, are NaN
  if (s_abort && tid == 0 && W.error) atomicCAS(W.error, 0u, kChunkError);
  if (s_abort && warp < 8) {
    const int i = warp >> 2, total = count_items(C, cu_q, kv_len, rows, R, small_rows);
    for (int k = item; k < s_claims; ++k) {
      const Item it = find_item(C, cu_q, kv_len, rows, R, small_rows, per, splits, total, longest, s_claimed[k & 3]);
      if (it.seq < 0) continue;
      const Row row = row_of(it, R, i, tid & 127);
      if (!row.live || it.z >= it.used) continue;
      for (int d = 0; d < D; ++d) out[(int64_t)row.tok * out_ld + (int64_t)row.h * D + d] = from_f32<O>(NAN);
      if (it.used > 1) {
        float* pp = part + (((int64_t)row.tok * heads + row.h) * splits + it.z) * (D + 8);
        for (int d = 0; d < D + 8; ++d) pp[d] = NAN;
      }
    }
  }
  if (warp == 8) {
    __syncwarp();
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
}

}  // namespace paged
}  // namespace le
