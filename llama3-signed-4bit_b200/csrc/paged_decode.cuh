// Decode form of llama_paged_attention: sequences of few new tokens (at most 16 query rows per kv
// head) over a long cache.
//
//   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  s_j = scale q . k_j,  m = max_j s_j
//
// in one pass with a running (m, l, o) per query row (a new maximum scales l and o by
// exp(m_old - m_new)).  Bound by the cache's bytes: 2 head_dim elements per key and kv head serve
// 4 G head_dim operations (G query heads share a kv head), far below the card's balance.
//
//   * The G heads x n tokens that share a kv head are the 16 rows of one mma.sync tile, so a key is
//     read once for all of them.  (The 5th-generation tensor cores would compute 128 rows of which
//     at most 16 exist; the product is a few per cent of the time either way.)
//   * The keys are cut into splits, one CTA each, and a CTA's four warps take
//     16-key slices of the split in turn.  A slice lies within one page (pages are multiples of
//     16 rows), so it has one table entry, and a page id out of range drops the slice.
//   * Every warp streams its slices through its own ring in shared memory (cp.async, 16-byte chunks
//     XOR-swizzled by row so that ldmatrix is free of conflicts): no barrier between the warps until
//     they merge their (m, l, o) at the end.  Rows past the length are zero-filled: what stale
//     memory holds there meets weights of 0 and must not be NaN.
//   * The splits of a sequence and kv head are one thread-block cluster where that suits the call: it cuts
//     the sequence evenly and joins the CTAs' unnormalised (m, l, o) through distributed shared
//     memory.  Otherwise they are written in fp32 and k_paged_combine joins them.  A sequence of one
//     split is written at once.
// The weights are rounded to the cache's type for the product with v (the type its v has), the sum
// l takes them unrounded in fp32.
//
// 128 sequences of up to 8192 keys, 8 kv heads of 128: 318 us, 2.07 GB at 6.5 TB/s, the rate of a plain
// copy.  64 of up to 2048, heads of 64: 34.6 us (140 MB; 21 us at that rate): the rest is the launches, the
// first loads (lengths, page, keys, one after the other), the last CTAs and the combine.  One sequence
// of 700 keys: 6.1 us, all latency.
#pragma once

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "paged.cuh"
#include "ptx.cuh"

namespace le {
namespace paged {

constexpr int kSlice = 16;        // keys a warp takes at a time
constexpr int kDecodeWarps = 4;
constexpr int kJoinSplits = 8;    // splits that a cluster joins at most
constexpr int kJoinKeys = 128;    // keys of such a split at least: two slices for each warp
template <int D> struct DecodeGeo {
  static constexpr int kStages = D == 64 ? 4 : 3;              // slices in flight per warp
  static constexpr int kSliceBytes = kSlice * D * 2;           // K (or V) of a slice
  static constexpr int kSmem = kDecodeWarps * kStages * 2 * kSliceBytes;
};

__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 16 bytes to shared memory, or zeros where !live (the source is not read then).
__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}

// Grid: seqs x splits x kv_heads, kv heads fastest (their CTAs read neighbouring bytes of the same
// rows); kJoin: seqs x kv_heads x splits, the splits of a pair a cluster.  per: keys of a split, a
// multiple of 64 (kJoin: of the sequence's own length); the last split takes all keys behind it.
// beside: launched while the chunk form of the same call runs, whose inputs are complete.
template <typename T, typename O, int D, bool kJoin>
__global__ void __launch_bounds__(32 * kDecodeWarps)
    k_paged_decode(Cache C, const T* __restrict__ q, int64_t q_ld, int heads, const int32_t* __restrict__ cu_q,
                   const int32_t* __restrict__ kv_len, int rows, float scale_log2, int per, int splits, int beside,
                   O* __restrict__ out, int64_t out_ld, float* __restrict__ part) {
  using Geo = DecodeGeo<D>;
  constexpr int kSt = Geo::kStages;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_m[kDecodeWarps][kDecodeRows], s_l[kDecodeWarps][kDecodeRows];
  grid_dep_launch();
  if (!beside) grid_dep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int z = kJoin ? blockIdx.x % splits : (blockIdx.x / C.kv_heads) % splits;
  const int g = (kJoin ? blockIdx.x / splits : blockIdx.x) % C.kv_heads;
  const int s = blockIdx.x / C.kv_heads / splits;
  const Span sp = span_of(C, cu_q, kv_len, s, rows);
  const int G = heads / C.kv_heads, R = sp.n * G;
  if (kJoin) per = max(kJoinKeys, ((sp.len + splits - 1) / splits + 63) & ~63);
  const int used = splits_of(sp.len, per, splits);
  namespace cg = cooperative_groups;
  if (sp.n <= 0 || R > kDecodeRows || z >= used) {  // nothing to do, or the chunk form's
    if (kJoin && sp.n > 0 && R <= kDecodeRows && used > 1) {  // the others of the cluster join
      cg::this_cluster().sync();
      cg::this_cluster().sync();
    }
    grid_dep_wait();
    return;
  }
  const int k0 = z * per, k1 = z == splits - 1 ? sp.len : min(sp.len, k0 + per);  // this split's keys

  // Q fragments: lane (r, c) = (lane / 4, lane % 4) holds rows r and r + 8
  const int fr = lane >> 2, fc = lane & 3;
  uint32_t qf[D / 16][4];
  {
    auto row_ptr = [&](int r) { return q + (int64_t)(sp.first + r / G) * q_ld + (int64_t)(g * G + r % G) * D + 2 * fc; };
    const T* q0 = row_ptr(min(fr, R - 1));
    const T* q1 = row_ptr(min(fr + 8, R - 1));
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      qf[k][0] = fr < R ? *reinterpret_cast<const uint32_t*>(q0 + 16 * k) : 0u;
      qf[k][1] = fr + 8 < R ? *reinterpret_cast<const uint32_t*>(q1 + 16 * k) : 0u;
      qf[k][2] = fr < R ? *reinterpret_cast<const uint32_t*>(q0 + 16 * k + 8) : 0u;
      qf[k][3] = fr + 8 < R ? *reinterpret_cast<const uint32_t*>(q1 + 16 * k + 8) : 0u;
    }
  }
  // last key of this lane's two rows
  const int lim0 = sp.len - sp.n + min(fr, R - 1) / G, lim1 = sp.len - sp.n + min(fr + 8, R - 1) / G;
  const bool upper = R > 8;

  // this warp's slices: slice i covers keys kw + 64 i ..
  const int kw = k0 + kSlice * warp;
  const int ns = k1 > kw ? (k1 - kw + 63) / 64 : 0;
  const uint32_t ring = smem_u32(smem) + (uint32_t)(warp * kSt * 2 * Geo::kSliceBytes);
  const int32_t* table = pages_of(C, s);
  const T* kp = static_cast<const T*>(C.k) + (int64_t)g * C.head_stride;
  const T* vp = static_cast<const T*>(C.v) + (int64_t)g * C.head_stride;
  int pages = -1;  // lane i: page of slice (block of 32) + i
  auto fetch_pages = [&](int i0) {
    const int j = kw + 64 * (i0 + lane);
    pages = i0 + lane < ns ? page_at(C, table, j >> C.page_log2) : -1;
  };
  auto load = [&](int i) {
    if (i < ns) {
      if ((i & 31) == 0) fetch_pages(i);
      const int page = __shfl_sync(0xffffffffu, pages, i & 31);
      if (page >= 0) {
        const int j = kw + 64 * i;
        const int64_t base = (int64_t)page * C.page_stride + (int64_t)(j & ((1 << C.page_log2) - 1)) * C.row_stride;
        const uint32_t st = ring + (uint32_t)((i % kSt) * 2 * Geo::kSliceBytes);
        constexpr int kCh = D / 8;  // 16-byte chunks of a row
#pragma unroll
        for (int x = 0; x < kSlice * kCh / 32; ++x) {
          const int r = (x * 32 + lane) / kCh, c = (x * 32 + lane) % kCh;
          const bool live = j + r < k1;
          const int64_t off = base + (int64_t)(live ? r : 0) * C.row_stride + 8 * c;
          const uint32_t d = st + (uint32_t)(r * D * 2 + ((c ^ (r & 7)) << 4));
          cp_async16_zfill(d, kp + off, live);
          cp_async16_zfill(d + Geo::kSliceBytes, vp + off, live);
        }
      }
    }
    cp_async_commit();  // one group per slice, empty ones included
  };
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.0f;
  unsigned live_pages = 0;  // bit i & 31: slice i has a page (set when its copies are issued)
  auto issue = [&](int i) {
    load(i);
    if (i < ns) {
      const bool ok = __shfl_sync(0xffffffffu, pages, i & 31) >= 0;
      live_pages = (live_pages & ~(1u << (i & 31))) | ((ok ? 1u : 0u) << (i & 31));
    }
  };
#pragma unroll
  for (int i = 0; i < kSt - 1; ++i) issue(i);
  for (int i = 0; i < ns; ++i) {
    issue(i + kSt - 1);
    cp_async_wait<kSt - 1>();
    __syncwarp();
    if ((live_pages >> (i & 31)) & 1u) {
      const uint32_t st = ring + (uint32_t)((i % kSt) * 2 * Geo::kSliceBytes);
      float c[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      const int kr = (lane & 7) + ((lane >> 4) << 3), kc = (lane >> 3) & 1;  // K: key row, 8-wide half
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        uint32_t b[4];
        ldsm4(st + (uint32_t)(kr * D * 2 + (((2 * k + kc) ^ (kr & 7)) << 4)), b);
        mma16816<T>(c[0], qf[k], b[0], b[1]);
        mma16816<T>(c[1], qf[k], b[2], b[3]);
      }
      const int j = kw + 64 * i;
      float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int key = j + 8 * h + 2 * fc + e;
          c[h][e] = key <= lim0 ? c[h][e] * scale_log2 : -INFINITY;
          t0 = fmaxf(t0, c[h][e]);
          if (upper) {
            c[h][2 + e] = key <= lim1 ? c[h][2 + e] * scale_log2 : -INFINITY;
            t1 = fmaxf(t1, c[h][2 + e]);
          }
        }
      t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 1));
      t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 2));
      if (upper) {
        t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 1));
        t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 2));
      }
      const float n0 = fmaxf(m0, t0), n1 = fmaxf(m1, t1);
      if (__any_sync(0xffffffffu, n0 > m0 || n1 > m1)) {
        // exp of a difference that would be inf - inf (no key yet) is taken as 1: l and o are 0
        const float a0 = n0 > m0 ? exp2_approx(m0 - n0) : 1.0f, a1 = n1 > m1 ? exp2_approx(m1 - n1) : 1.0f;
        l0 *= a0;
        l1 *= a1;
#pragma unroll
        for (int x = 0; x < D / 8; ++x) {
          o[x][0] *= a0; o[x][1] *= a0;
          o[x][2] *= a1; o[x][3] *= a1;
        }
        m0 = n0;
        m1 = n1;
      }
      const float z0 = m0 == -INFINITY ? 0.0f : m0, z1 = m1 == -INFINITY ? 0.0f : m1;
      uint32_t p[4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float e0 = exp2_approx(c[h][0] - z0), e1 = exp2_approx(c[h][1] - z0);
        l0 += e0 + e1;
        p[2 * h] = pack2<T>(e0, e1);
        p[2 * h + 1] = 0u;
        if (upper) {
          const float f0 = exp2_approx(c[h][2] - z1), f1 = exp2_approx(c[h][3] - z1);
          l1 += f0 + f1;
          p[2 * h + 1] = pack2<T>(f0, f1);
        }
      }
      const int vr = (lane & 7) + (((lane >> 3) & 1) << 3), vc = lane >> 4;  // V: key row, 8-wide half
#pragma unroll
      for (int x = 0; x < D / 16; ++x) {
        uint32_t b[4];
        ldsm4t(st + Geo::kSliceBytes + (uint32_t)(vr * D * 2 + (((2 * x + vc) ^ (vr & 7)) << 4)), b);
        mma16816<T>(o[2 * x], p, b[0], b[1]);
        mma16816<T>(o[2 * x + 1], p, b[2], b[3]);
      }
    }
    __syncwarp();  // the slot is free for slice i + kSt
  }
  cp_async_wait<0>();
  l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
  l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
  l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
  l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
  // merge of the four warps: their o rows through shared memory (the rings are done with)
  __syncthreads();
  float* so = reinterpret_cast<float*>(smem);  // [warp][row][D]
  if (fc == 0) {
    s_m[warp][fr] = m0; s_l[warp][fr] = l0;
    s_m[warp][fr + 8] = m1; s_l[warp][fr + 8] = l1;
  }
#pragma unroll
  for (int x = 0; x < D / 8; ++x) {
    *reinterpret_cast<float2*>(&so[(warp * kDecodeRows + fr) * D + 8 * x + 2 * fc]) = make_float2(o[x][0], o[x][1]);
    if (upper)
      *reinterpret_cast<float2*>(&so[(warp * kDecodeRows + fr + 8) * D + 8 * x + 2 * fc]) = make_float2(o[x][2], o[x][3]);
  }
  __syncthreads();
  constexpr int kPer = 8;  // elements a thread merges at a time
  constexpr int kItems = kDecodeRows * D / kPer / (32 * kDecodeWarps);  // of them at most
  const int items = R * (D / kPer);
  auto finish = [&](int i, float L, float (&a)[kPer]) {
    const float inv = L > 0.0f ? 1.0f / L : 0.0f;  // no key: zeros
#pragma unroll
    for (int e = 0; e < kPer; ++e) a[e] *= inv;
    const int r = i / (D / kPer);
    store8(out + (int64_t)(sp.first + r / G) * out_ld + (int64_t)(g * G + r % G) * D + i % (D / kPer) * kPer, a);
  };
  float M[kItems], L[kItems], a[kItems][kPer];
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    const int i = threadIdx.x + k * 32 * kDecodeWarps, r = i / (D / kPer), d = i % (D / kPer) * kPer;
    if (i >= items) break;
    M[k] = s_m[0][r];
#pragma unroll
    for (int w = 1; w < kDecodeWarps; ++w) M[k] = fmaxf(M[k], s_m[w][r]);
    L[k] = 0.0f;
#pragma unroll
    for (int e = 0; e < kPer; ++e) a[k][e] = 0.0f;
#pragma unroll
    for (int w = 0; w < kDecodeWarps; ++w) {
      const float f = s_m[w][r] == -INFINITY ? 0.0f : exp2_approx(s_m[w][r] - M[k]);
      L[k] = fmaf(s_l[w][r], f, L[k]);
#pragma unroll
      for (int e = 0; e < kPer; ++e) a[k][e] = fmaf(so[(w * kDecodeRows + r) * D + d + e], f, a[k][e]);
    }
    if (used == 1) finish(i, L[k], a[k]);
    else if (!kJoin) write_part<D>(part, (((int64_t)s * C.kv_heads + g) * kDecodeRows + r) * splits + z, d, M[k], L[k], a[k]);
  }
  if (kJoin && used > 1) {
    cg::cluster_group cl = cg::this_cluster();
    __syncthreads();  // the warps' o have been read: the CTA's own goes over them, row by row as in a part
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const int i = threadIdx.x + k * 32 * kDecodeWarps;
      if (i < items) write_part<D>(so, i / (D / kPer), i % (D / kPer) * kPer, M[k], L[k], a[k]);
    }
    cl.sync();
    for (int i = threadIdx.x + 32 * kDecodeWarps * z; i < items; i += 32 * kDecodeWarps * used) {
      const int r = i / (D / kPer), d = i % (D / kPer) * kPer;
      float2 ml[kJoinSplits];
      float m = -INFINITY, l = 0.0f, x[kPer] = {};
#pragma unroll
      for (int y = 0; y < kJoinSplits; ++y) {
        ml[y] = y < used ? *reinterpret_cast<const float2*>(cl.map_shared_rank(so, y) + r * (D + 8) + D)
                         : make_float2(-INFINITY, 0.0f);
        m = fmaxf(m, ml[y].x);
      }
#pragma unroll
      for (int y = 0; y < kJoinSplits; ++y) {
        if (y >= used) break;
        const float f = ml[y].x == -INFINITY ? 0.0f : exp2_approx(ml[y].x - m);
        float v[kPer];
        load8(cl.map_shared_rank(so, y) + r * (D + 8) + d, v);
        l = fmaf(ml[y].y, f, l);
#pragma unroll
        for (int e = 0; e < kPer; ++e) x[e] = fmaf(v[e], f, x[e]);
      }
      finish(i, l, x);
    }
    cl.sync();  // nobody's shared memory goes before it has been read
  }
  // launched beside the chunk form: this grid ends after it, so that whoever waits for this one
  // has waited for both
  grid_dep_wait();
}

}  // namespace paged
}  // namespace le
