// Chunk form of llama_paged_attention: prompt chunks of any length over the paged cache, on the
// tcgen05 tensor cores.
//
//   o = sum_j 2^(c s_j - c m) v_j / sum_j 2^(c s_j - c m),  s_j = q . k_j,  c = scale log2(e)
//
// The G query heads that share a kv head and the n tokens of a sequence form one axis of n G rows
// (token-major), cut into work items of 256 rows = two MMA tiles of 128; every key is read once
// for all 256.  One CTA (one per SM) takes an item and walks its keys in tiles of 128:
//
//   * warp 9 brings the K and V rows of a tile into a ring of shared-memory stages by TMA, one box
//     per page and 64-element column block, straight into the 128-byte-swizzled layouts that the
//     MMA reads: K as the K-major operand of S = Q K^T, V (whose rows are keys) as the MN-major
//     operand of O += P V, so nothing is transposed.  Pages past the keys, and page ids out of range,
//     are addressed past the pool's last page: TMA fills them with zeros.  The rows of the last page
//     behind the length may hold anything, NaN too, which a weight of 0 would not silence: the
//     loader zeroes them in its V stage and releases that tile's product by a barrier of its own.
//   * warp 8 (one thread) issues the products, alternating between the two row tiles so that one
//     tile's products run while the other's softmax does: P_i V_j, then S_i of the next key tile.
//     S_i (128 fp32 columns of tensor memory) is overwritten in place by P_i (64 columns), O_i
//     accumulates in D columns.
//   * warps 0..3 and 4..7 are the softmax of tile 0 and 1, a thread per row (= tensor-memory lane), so
//     that a row's maximum and sum need no exchange.  O is only rescaled when a row's maximum has
//     grown by more than 2^8 since the value it is scaled by; until then weights may exceed 1, by at
//     most 2^8, which costs no accuracy in fp32 sums or 16-bit weights.
// Weights are rounded to the cache's type as the A operand of P V; their sum is taken in fp32 before
// that.  Bound by the products for head_dim 128 and by the exponentials (16 a clock and SM) for 64.
//
// All mbarrier waits are bounded; on timeout the error word is set, every role stops, the copies and
// products in flight are waited for (again bounded) and the item's rows become NaN.
#pragma once

#include <cuda.h>

#include "ops.h"
#include "paged.cuh"
#include "ptx.cuh"

namespace le {
namespace paged {

constexpr int kTileRows = 128;                 // rows of an MMA tile
constexpr int kItemRows = 2 * kTileRows;
constexpr int kTileKeys = 128;
constexpr int kChunkThreads = 320;
constexpr int kBlockBytes = kTileKeys * 128;   // one 64-element column block of 128 rows
constexpr float kLazyLog2 = 8.0f;              // growth of a maximum that forces a rescale (log2)
template <int D> struct ChunkGeo {
  static constexpr int kCols = D / 64;                       // column blocks of a row
  static constexpr int kStageBytes = kCols * kBlockBytes;    // K or V of a key tile
  static constexpr int kStages = D == 64 ? 8 : 5;
  static constexpr int kQBytes = 2 * kStageBytes;
  static constexpr int kSmem = 1024 + kQBytes + kStages * kStageBytes;
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
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
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

// Waits (bounded) for phase `parity`; false after a timeout here or elsewhere in the CTA.
__device__ __forceinline__ bool chunk_wait(uint32_t bar, uint32_t parity, volatile uint32_t* abort, const Waits& W) {
  if (mbar_try(bar, parity)) return true;
  const unsigned long long t0 = gtimer();
  while (!mbar_try_sleep(bar, parity, 20000)) {
    if (*abort) return false;
    if (gtimer() - t0 > W.ns) {
      *abort = 1u;
      atomicCAS(W.error, 0u, kChunkError);
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ void chunk_drain(uint32_t bar, uint32_t parity, const Waits& W) {
  const unsigned long long t0 = gtimer();
  while (!mbar_try_sleep(bar, parity, 20000) && gtimer() - t0 < W.ns) {
  }
}

// Grid: items x splits x kv_heads (kv heads fastest), items >= the sum over sequences of
// ceil(n G / 256); the last items (the longest of each sequence) come first.  per: keys of a split,
// a multiple of 128.  Sequences of at most small_rows rows per kv head are the decode form's.
template <typename T, typename O, int D>
__global__ void __launch_bounds__(kChunkThreads, 1)
    k_paged_chunk(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, Cache C,
                  const T* __restrict__ q, int64_t q_ld, int heads, const int32_t* __restrict__ cu_q,
                  const int32_t* __restrict__ kv_len, int rows, float scale, int small_rows, int per, int splits,
                  O* __restrict__ out, int64_t out_ld, float* __restrict__ part, Waits W) {
  using Geo = ChunkGeo<D>;
  constexpr int kSt = Geo::kStages;
  extern __shared__ uint8_t chunk_smem[];
  __shared__ __align__(8) unsigned long long s_bar[2 * kSt + 7];
  __shared__ uint32_t s_tmem;
  __shared__ volatile uint32_t s_abort;
  __shared__ int s_item[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  grid_dep_wait();
  grid_dep_launch();  // the decode form of the same call may start: its inputs are complete
  const int G = heads / C.kv_heads;
  const int g = blockIdx.x % C.kv_heads;
  const int z = (blockIdx.x / C.kv_heads) % splits;
  if (warp == 0) {
    // the work item: count every sequence's items, then find the one that holds ours from the end
    auto items_of = [&](int s) {
      if (s >= C.seqs) return 0;
      const Span x = span_of(C, cu_q, kv_len, s, rows);
      const int r = max(x.n, 0) * G;
      return r <= small_rows ? 0 : (r + kItemRows - 1) / kItemRows;
    };
    int total = 0;
    for (int s0 = 0; s0 < C.seqs; s0 += 32) total += items_of(s0 + lane);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    const int want = total - 1 - blockIdx.x / C.kv_heads / splits;
    int before = 0, seq = -1, item = 0;
    for (int s0 = 0; s0 < C.seqs && seq < 0 && want >= 0; s0 += 32) {
      const int mine = items_of(s0 + lane);
      int inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + inc > want);
      if (hit) {
        const int l = __ffs(hit) - 1;
        seq = s0 + l;
        item = want - before - __shfl_sync(0xffffffffu, inc - mine, l);
      }
      before += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (lane == 0) {
      s_item[0] = seq;
      s_item[1] = item;
      s_abort = 0u;
      // full[st] 0.., empty[st] kSt.., S ready (2), P ready (2), O done (2), V tail zeroed
      for (int i = 0; i < 2 * kSt + 7; ++i) {
        const bool p = i == 2 * kSt + 2 || i == 2 * kSt + 3;
        mbar_init(smem_u32(&s_bar[i]), p ? kTileRows : 1);
      }
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
  }
  __syncthreads();
  const int s = s_item[0];
  const Span sp = s >= 0 ? span_of(C, cu_q, kv_len, s, rows) : Span{0, 0, 0};
  const int used = splits_of(sp.len, per, splits);
  if (s < 0 || z >= used) return;  // uniform over the CTA, before any tensor memory is held
  const int R = sp.n * G;                              // rows of the sequence for this kv head
  const int row0 = s_item[1] * kItemRows;              // first of this item
  const int shift = sp.len - sp.n;                     // position of token 0
  // keys of a tile's rows: all up to its last row's position, within this split
  const int k_lo = z * per;
  auto keys_end = [&](int i) {
    const int r_last = min(row0 + (i + 1) * kTileRows, R) - 1;
    if (r_last < row0 + i * kTileRows) return 0;
    const int e = min(sp.len, shift + r_last / G + 1);
    return z == splits - 1 ? e : min(e, k_lo + per);
  };
  auto tiles_to = [&](int end) { return end > k_lo ? (end - k_lo + kTileKeys - 1) / kTileKeys : 0; };
  const int nk0 = tiles_to(keys_end(0)), nk1 = tiles_to(keys_end(1));
  const int nk = max(nk0, nk1);
  const int32_t* table = pages_of(C, s);
  const int page_mask = (1 << C.page_log2) - 1;
  const int k_hi = min(sp.len, k_lo + nk * kTileKeys);  // keys that are loaded

  const uint32_t base = (smem_u32(chunk_smem) + 1023u) & ~1023u;
  const uint32_t stage0 = base + Geo::kQBytes;
  auto bar = [&](int i) { return smem_u32(&s_bar[i]); };
  const int kBarS = 2 * kSt, kBarP = 2 * kSt + 2, kBarO = 2 * kSt + 4, kBarFix = 2 * kSt + 6;
  if (warp == 8) {
    tc::tmem_alloc(smem_u32(&s_tmem), 512);
    tc::tmem_relinquish();
  }
  // are all of the item's pages valid?  (a table that holds bad ids costs a check per tile)
  bool bad = false;
  for (int e = (k_lo >> C.page_log2) + tid; e <= ((k_hi - 1) >> C.page_log2) && k_hi > k_lo; e += kChunkThreads) {
    bad |= page_at(C, table, e) < 0;
  }
  // Q rows into the K-major swizzled layout: tile i, column block, 128 rows of 128 bytes; a negative
  // scale is moved into q, so that the maximum of s is that of scale s
  const uint32_t flip = scale < 0.0f ? 0x80008000u : 0u;
  for (int i = tid; i < kItemRows * (D / 8); i += kChunkThreads) {
    const int r = i / (D / 8), ch = i % (D / 8);
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (row0 + r < R) {
      const int tok = (row0 + r) / G, h = g * G + (row0 + r) % G;
      v = *reinterpret_cast<const uint4*>(q + (int64_t)(sp.first + tok) * q_ld + (int64_t)h * D + 8 * ch);
      v.x ^= flip; v.y ^= flip; v.z ^= flip; v.w ^= flip;
    }
    const uint32_t a = base + (uint32_t)((r >> 7) * Geo::kStageBytes + (ch >> 3) * kBlockBytes + (r & 127) * 128 +
                                         (((ch & 7) ^ (r & 7)) << 4));
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  tc::tc_fence_before();
  const bool any_bad = __syncthreads_or(bad ? 1 : 0) != 0;
  tc::tc_fence_after();
  const uint32_t tmem = s_tmem;
  // a tile that reaches past the length shares its last page with rows that hold anything
  const int fix_tile = (sp.len & page_mask) != 0 && k_lo + nk * kTileKeys > sp.len ? nk - 1 : -1;

  if (warp == 9) {
    // ---- loader ----
    const int box = min(1 << C.page_log2, kTileKeys), boxes = kTileKeys / box;
    bool ok = true;
    int fills = 0;
    auto page_of = [&](int j) {  // this lane's page of tile j; none: behind the pool's last
      const int key = k_lo + j * kTileKeys + lane * box;
      const int p = lane < boxes && key < k_hi ? page_at(C, table, key >> C.page_log2) : -1;
      return p >= 0 ? p : C.num_pages;
    };
    int page = page_of(0);
    for (int j = 0; j < nk && ok; ++j) {
      const int next = j + 1 < nk ? page_of(j + 1) : 0;
      const int row = (k_lo + j * kTileKeys) & page_mask;  // nonzero only where pages exceed a tile
      for (int v = 0; v < 2 && ok; ++v) {
        const int st = fills % kSt;
        if (fills >= kSt) ok = __all_sync(0xffffffffu, chunk_wait(bar(kSt + st), (uint32_t)(fills / kSt - 1) & 1u, &s_abort, W));
        if (!ok) break;
        if (lane == 0) mbar_expect_tx(bar(st), Geo::kStageBytes);
        __syncwarp();
        if (lane < boxes) {
#pragma unroll
          for (int cb = 0; cb < Geo::kCols; ++cb)
            tma_box(stage0 + (uint32_t)(st * Geo::kStageBytes + cb * kBlockBytes + lane * box * 128), v ? &map_v : &map_k,
                    cb * 64, g, row, page, bar(st));
        }
        ++fills;
        if (v == 1 && j == fix_tile) {
          ok = __all_sync(0xffffffffu, chunk_wait(bar(st), (uint32_t)((fills - 1) / kSt) & 1u, &s_abort, W));
          const int r0 = sp.len - (k_lo + j * kTileKeys);  // first row behind the length
          for (int i = lane; i < (kTileKeys - r0) * 8 * Geo::kCols; i += 32) {
            const int cb = i / ((kTileKeys - r0) * 8), x = i % ((kTileKeys - r0) * 8);
            const uint32_t a = stage0 + (uint32_t)(st * Geo::kStageBytes + cb * kBlockBytes + r0 * 128 + x * 16);
            asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(a), "r"(0u) : "memory");
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0 && ok) mbar_arrive_n(bar(kBarFix), 1);
        }
      }
      page = next;
    }
    if (s_abort)  // the copies in flight land before the shared memory goes
      for (int f = max(0, fills - kSt); f < fills; ++f) chunk_drain(bar(f % kSt), (uint32_t)(f / kSt) & 1u, W);
  } else if (warp == 8) {
    // ---- products ----
    if (lane == 0) {
      constexpr uint32_t id_s = chunk_idesc<T>(kTileKeys, 0), id_o = chunk_idesc<T>(D, 1);
      bool ok = true;
      int last = -1, last_parity = 0;
      auto commit = [&](int b, int n) {  // n: how often this barrier was committed before
        tc::tc_commit(bar(b));
        last = b;
        last_parity = n & 1;
      };
      auto wait = [&](int b, int n) { return chunk_wait(bar(b), (uint32_t)n & 1u, &s_abort, W); };
      // S_i of key tile j, from fill 2 j of the ring
      auto issue_s = [&](int i, int j) {
        const uint32_t a = base + (uint32_t)(i * Geo::kStageBytes), b = stage0 + (uint32_t)((2 * j % kSt) * Geo::kStageBytes);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = (uint32_t)((k >> 2) * kBlockBytes);
          chunk_mma_ss(tmem + 128u * i, tc::sw128_desc(a + off) + 2 * (k & 3), tc::sw128_desc(b + off) + 2 * (k & 3), id_s,
                       k > 0 ? 1u : 0u);
        }
        commit(kBarS + i, j);
      };
      auto full = [&](int f) { return wait(f % kSt, f / kSt); };
      auto free_stage = [&](int f) { commit(kSt + f % kSt, f / kSt); };
      if (W.expire) ok = wait(kBarO, 0);  // test only: no product has been issued, so the wait runs out
      if (ok && nk > 0 && (ok = full(0))) {
        tc::tc_fence_after();
        if (nk0 > 0) issue_s(0, 0);
        if (nk1 > 0) issue_s(1, 0);
        free_stage(0);
      }
      for (int j = 0; j < nk && ok; ++j) {
        const int fv = 2 * j + 1;
        ok = full(fv) && (j != fix_tile || wait(kBarFix, 0));
        const uint32_t v = stage0 + (uint32_t)((fv % kSt) * Geo::kStageBytes);
        bool next = false;  // K of the next tile has landed
        for (int i = 0; i < 2 && ok; ++i) {
          if (j >= (i ? nk1 : nk0)) continue;
          ok = wait(kBarP + i, j);
          if (!ok) break;
          tc::tc_fence_after();
#pragma unroll
          for (int k = 0; k < kTileKeys / 16; ++k)  // 16 keys: 8 columns of P, 2048 bytes of V
            tc::tc_mma_ts(tmem + 256u + 128u * i, tmem + 128u * i + 8u * k, mn_desc(v + 2048u * k), id_o,
                          (j > 0 || k > 0) ? 1u : 0u);
          commit(kBarO + i, j);
          if (j + 1 < (i ? nk1 : nk0)) {
            if (!next) ok = full(2 * j + 2);
            next = true;
            if (!ok) break;
            tc::tc_fence_after();
            issue_s(i, j + 1);
          }
        }
        if (ok) {
          free_stage(fv);
          if (j + 1 < nk) free_stage(2 * j + 2);
        }
      }
      if (s_abort && last >= 0) chunk_drain(bar(last), (uint32_t)last_parity, W);
    }
    __syncwarp();
  } else {
    // ---- softmax of tile i, a thread per row ----
    const int i = warp >> 2;
    const int nki = i ? nk1 : nk0;
    const int r = row0 + i * kTileRows + (tid & 127);
    const int rc = min(r, R - 1);  // rows past the end see what the last one does
    const int lim = shift + rc / G;
    const int lim_first = shift + (row0 + i * kTileRows) / G;
    const float c = fmaxf(fabsf(scale) * 1.44269504f, 1e-30f);  // > 0: a masked -inf stays -inf
    const uint32_t t_s = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + 128u * i;
    const uint32_t t_o = t_s - 128u * i + 256u + 128u * i;
    float m = -INFINITY, l[2] = {0.0f, 0.0f};  // the maximum that O and l are scaled by; the sum's two halves
    bool ok = true;
    for (int j = 0; j < nki; ++j) {
      ok = __all_sync(0xffffffffu, chunk_wait(bar(kBarS + i), (uint32_t)j & 1u, &s_abort, W));
      if (!ok) break;
      tc::tc_fence_after();
      uint32_t u[4][32];  // the row's 128 scores
#pragma unroll
      for (int x = 0; x < 4; ++x) tc::tmem_ld32(t_s + 32u * x, u[x]);
      tc::tmem_wait_ld();
      const int key0 = k_lo + j * kTileKeys;
      if (key0 + kTileKeys - 1 > lim_first) {
        const int rel = lim - key0;
#pragma unroll
        for (int x = 0; x < kTileKeys; ++x) u[x >> 5][x & 31] = x <= rel ? u[x >> 5][x & 31] : kNegInf;
      }
      if (any_bad) {  // bit x: the tile's keys 16 x .. 16 x + 15 have a page
        const int key = key0 + 16 * (lane & 7);
        const unsigned live = __ballot_sync(0xffffffffu, key < sp.len && page_at(C, table, key >> C.page_log2) >= 0);
#pragma unroll
        for (int x = 0; x < kTileKeys; ++x) u[x >> 5][x & 31] = (live >> (x / 16)) & 1u ? u[x >> 5][x & 31] : kNegInf;
      }
      // maximum, as four chains of three-operand maxima
      float mx[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        mx[x] = max3(__uint_as_float(u[x][0]), __uint_as_float(u[x][1]), __uint_as_float(u[x][2]));
#pragma unroll
        for (int e = 3; e < 31; e += 2) mx[x] = max3(mx[x], __uint_as_float(u[x][e]), __uint_as_float(u[x][e + 1]));
      }
      float mt = max3(mx[0], mx[1], mx[2]);
      mt = max3(mt, mx[3], __uint_as_float(u[0][31]));
      mt = max3(mt, __uint_as_float(u[1][31]), __uint_as_float(u[2][31]));
      mt = fmaxf(mt, __uint_as_float(u[3][31]));
      const bool grow = j == 0 ? mt > m : (mt - m) * c > kLazyLog2;
      if (__any_sync(0xffffffffu, grow)) {
        const float alpha = grow ? exp2_approx((m - mt) * c) : 1.0f;
        m = grow ? mt : m;
        l[0] *= alpha;
        l[1] *= alpha;
        if (j > 0) {
          ok = __all_sync(0xffffffffu, chunk_wait(bar(kBarO + i), (uint32_t)(j - 1) & 1u, &s_abort, W));
          if (!ok) break;
          tc::tc_fence_after();
#pragma unroll
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
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        uint32_t p[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float2 y = fma2(make_float2(__uint_as_float(u[x][2 * e]), __uint_as_float(u[x][2 * e + 1])), c2, mc2);
          y.x = exp2_approx(y.x);
          y.y = exp2_approx(y.y);
          if (e & 1) sum1 = add2(sum1, y);
          else sum0 = add2(sum0, y);
          p[e] = pack2<T>(y.x, y.y);
        }
        tmem_st16<16>(t_s + 16u * x, p);
      }
      l[0] += sum0.x + sum1.x;
      l[1] += sum0.y + sum1.y;
      tc::tmem_wait_st();
      tc::tc_fence_before();
      mbar_arrive_n(bar(kBarP + i), 1);
    }
    if (ok && nki > 0) {
      ok = __all_sync(0xffffffffu, chunk_wait(bar(kBarO + i), (uint32_t)(nki - 1) & 1u, &s_abort, W));
      tc::tc_fence_after();
    }
    // ---- result: the row's D outputs, or this split's part of them ----
    const int tok = sp.first + rc / G, h = g * G + rc % G;
    const float sum = l[0] + l[1], inv = !ok ? NAN : sum > 0.0f ? 1.0f / sum : 0.0f;
    float* pp = part + (((int64_t)tok * heads + h) * splits + z) * (D + 8);
    O* po = out + (int64_t)tok * out_ld + (int64_t)h * D;
#pragma unroll
    for (int x = 0; x < D / 32; ++x) {
      uint32_t v[32];
#pragma unroll
      for (int e = 0; e < 32; ++e) v[e] = 0u;
      if (nki > 0 && ok) {
        tc::tmem_ld32(t_o + 32u * x, v);
        tc::tmem_wait_ld();
      }
      if (r < R) {
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          float a[8];
#pragma unroll
          for (int y = 0; y < 8; ++y) a[y] = __uint_as_float(v[e + y]);
          if (used > 1) {
            store8(pp + 32 * x + e, a);
          } else {
#pragma unroll
            for (int y = 0; y < 8; ++y) a[y] *= inv;
            store8(po + 32 * x + e, a);
          }
        }
      }
    }
    if (r < R && used > 1)
      *reinterpret_cast<float2*>(pp + D) = ok ? make_float2(m == -INFINITY ? m : m * c, sum) : make_float2(0.0f, NAN);
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    __syncwarp();
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
}

}  // namespace paged
}  // namespace le
