"""llama_paged_append and llama_paged_attention against the formulas in 64 bits.

Tolerances.  With h = finfo(type).eps / 2 (half a step, relative):
* append: the rotation is two fp32 products and a sum (each off by at most 2^-24 of its result, so
  together by 2^-23 (|x c| + |y s|)), then one rounding to the output type, h |r|, or half the
  smallest subnormal where r is below the type's normal range.
* attention: every softmax weight is rounded to the cache's type before it meets v, which moves an
  output by at most h sum_j p_j |v_j|; weights below fp16's normal range round absolutely, by at most
  2^-25 each against a sum of at least 1 (N 2^-25 max |v|).  A score q . k carries at most
  (D + 4) 2^-24 scale sum |q_i k_i| of fp32 error and the exponential 2^-20 relative, which moves each
  weight by that much relative and the output by twice that times sum p |v| (numerator and sum);
  fp32 accumulation over N keys adds at most 2 N 2^-24 of it.  Then the output's own rounding, h |o|.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib(pkg, gpu_available):
    return pkg.LlamaEngineBindings().lib


def codes(pkg):
    import torch
    return {torch.float32: pkg.F32, torch.float16: pkg.F16, torch.bfloat16: pkg.BF16}


class Pool:
    """A paged cache with a shuffled table; unused rows hold NaN, as stale memory may."""

    def __init__(self, pkg, dtype, kv_heads, d, page, lens, seed, head_major=False, spare=3, layers=1, layer=0):
        import torch
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        need = [(n + page - 1) // page for n in lens]
        self.width = max(1, max(need)) + 1
        total = sum(need) + spare
        perm = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
        self.table = torch.full((len(lens), self.width + 2), -7, dtype=torch.int32, device="cuda")
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = perm[at:at + n]
            at += n
        shape = (total, layers, kv_heads, page, d) if head_major else (total, layers, page, kv_heads, d)
        full = [torch.full(shape, float("nan"), dtype=dtype, device="cuda") for _ in range(2)]
        # views [page][row][head][d]
        self.k, self.v = [(t[:, layer].permute(0, 2, 1, 3) if head_major else t[:, layer]) for t in full]
        self.page, self.kv_heads, self.d, self.dtype, self.total = page, kv_heads, d, dtype, total
        self.desc = pkg.PagedKV(k=self.k.data_ptr(), v=self.v.data_ptr(), type=codes(pkg)[dtype], num_pages=total,
                                page_size=page, kv_heads=kv_heads, head_dim=d, page_stride=self.k.stride(0),
                                row_stride=self.k.stride(1), head_stride=self.k.stride(2), table=self.table.data_ptr(),
                                table_stride=self.table.stride(0), table_width=self.width, seqs=len(lens))
        self.gen = g

    def fill(self, lens, scale=1.0):
        """Random keys and values for the first lens[s] keys of every sequence."""
        import torch
        for s, n in enumerate(lens):
            pg, sl = self.where(s, torch.arange(n, device="cuda"))
            for t in (self.k, self.v):
                x = torch.randn((n, self.kv_heads, self.d), generator=self.gen, device="cuda") * scale
                t[pg, sl] = x.to(self.dtype)

    def where(self, s, pos):
        return self.table[s].long()[pos // self.page], pos % self.page

    def rows(self, s, n):
        import torch
        pg, sl = self.where(s, torch.arange(n, device="cuda"))
        return self.k[pg, sl].double(), self.v[pg, sl].double()


def attend(pkg, lib, pool, q, heads, news, lens, out, max_q=None, max_kv=None, rows=None, scale=None, stream=0):
    import torch
    cu = torch.tensor(np.cumsum([0] + list(news)), dtype=torch.int32, device="cuda")
    kvl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    rows = q.shape[0] if rows is None else rows
    max_q = max(news) if max_q is None else max_q
    max_kv = max(lens) if max_kv is None else max_kv
    size = lib.llama_paged_attention_workspace(ctypes.byref(pool.desc), heads, rows, max_q, max_kv)
    ws = torch.full((size + 16,), 255, dtype=torch.uint8, device="cuda")  # NaN patterns: nothing may rely on it
    scale = pool.d ** -0.5 if scale is None else scale
    rc = lib.llama_paged_attention(ctypes.byref(pool.desc), q.data_ptr(), q.stride(0), heads, cu.data_ptr(), kvl.data_ptr(),
                                   rows, max_q, max_kv, scale, out.data_ptr(), codes(pkg)[out.dtype], out.stride(0),
                                   ws.data_ptr(), size, stream)
    assert rc == 0, lib.llama_engine_last_error(None)
    assert bool((ws[size:] == 255).all())
    return cu, kvl, ws


def check_attention(pool, q, heads, news, lens, out, scale=None, dead=None):
    """Every output row against the formula in 64 bits, element by element; dead[s]: keys left out."""
    import torch
    d, kvh = pool.d, pool.kv_heads
    g = heads // kvh
    scale = d ** -0.5 if scale is None else scale
    h = torch.finfo(pool.dtype).eps / 2
    ho = torch.finfo(out.dtype).eps / 2
    at = 0
    for s, (n, kv) in enumerate(zip(news, lens)):
        if n == 0:
            continue
        k, v = pool.rows(s, kv) if kv else (torch.zeros((0, kvh, d), device="cuda").double(),) * 2
        qq = q[at:at + n].double().view(n, kvh, g, d)
        seen = torch.arange(kv, device="cuda")[None, :] <= torch.arange(kv - n, kv, device="cuda")[:, None]
        if dead and s in dead:
            seen[:, dead[s]] = False
            k, v = torch.nan_to_num(k), torch.nan_to_num(v)
        e = torch.einsum("thgd,khd->hgtk", qq, k) * scale
        e = e.masked_fill(~seen, -math.inf)
        top = e.amax(dim=-1, keepdim=True) if kv else torch.zeros((kvh, g, n, 1), device="cuda").double()
        p = torch.where(seen, torch.exp(e - top), 0.0)
        z = p.sum(dim=-1, keepdim=True)
        p = torch.where(z > 0, p / z, 0.0)
        ref = torch.einsum("hgtk,khd->thgd", p, v).reshape(n, heads * d)
        mag = torch.einsum("hgtk,khd->thgd", p, v.abs()).reshape(n, heads * d)
        err_s = (d + 4) * 2.0 ** -24 * scale * (torch.einsum("thgd,khd->hgtk", qq.abs(), k.abs()).amax().item() if kv else 0)
        rel = h + 2 * (err_s + 2.0 ** -20) + 2 * kv * 2.0 ** -24
        tol = rel * mag + ho * ref.abs() + (kv * 2.0 ** -25 * v.abs().amax().item() if kv else 0) + 1e-30
        got = out[at:at + n].double()
        bad = ~((got - ref).abs() <= tol)
        assert not bool(bad.any()), (s, n, kv, int(bad.sum()), (got - ref).abs().max().item(), bad.nonzero()[:4].tolist())
        at += n


SHAPES = [
    # dtype, head_dim, heads, kv_heads, page, new tokens, keys
    ("f16", 64, 32, 8, 16, [1], [700]),
    ("f16", 64, 32, 8, 16, [1], [1]),
    ("bf16", 128, 8, 1, 32, [1, 1, 1], [64, 65, 63]),
    ("f16", 64, 4, 4, 16, [1, 0, 1, 1, 1], [17, 40, 0, 128, 1023]),           # an idle sequence, one without keys
    ("bf16", 128, 28, 4, 64, [1] * 9, [1, 16, 31, 129, 257, 700, 2049, 4000, 5]),
    ("f16", 64, 32, 8, 16, [5, 3, 2], [5, 300, 2]),
    ("f16", 64, 32, 8, 16, [128], [128]),
    ("f16", 64, 32, 8, 256, [129], [1000]),
    ("bf16", 64, 6, 2, 16, [63, 1, 200, 7], [63, 500, 333, 8]),
    ("bf16", 128, 32, 8, 16, [257], [777]),
    ("f16", 128, 28, 4, 32, [1, 37, 1, 300, 0, 2], [900, 37, 1, 1301, 50, 130]),
    ("bf16", 128, 5, 5, 128, [600], [600]),
    ("f16", 64, 64, 1, 16, [1, 3], [130, 4]),                                    # one kv head for all
    ("bf16", 128, 16, 8, 64, [4, 70], [2, 30]),                                  # more tokens than keys: empty rows
    ("f16", 128, 160, 1, 16, [1, 9], [1000, 260]),                               # more heads per kv head than a tile's rows
    ("f16", 64, 32, 8, 64, [300, 300], [4096, 301]),
    ("bf16", 128, 32, 8, 64, [20], [9000]),                                      # few rows, a long cache: split and joined
    # many items for every SM: odd numbers of row tiles, tiles without keys, splits that end early, tails
    ("bf16", 128, 28, 4, 16, [33, 1, 19, 200, 0, 37, 18, 36, 55, 90, 1, 130, 17, 300, 64, 5] * 4,
     [40, 9, 21, 1999, 3, 37, 333, 36, 60, 1500, 1, 130, 18, 311, 64, 7] * 4),
    ("f16", 64, 12, 2, 32, [33, 7, 100, 200, 1, 37, 64, 21, 43, 90, 11, 130, 17, 300] * 6,
     [33, 5, 4000, 201, 9, 37, 64, 400, 44, 3, 1100, 130, 18, 311] * 6),
    ("f16", 128, 200, 1, 16, [1, 2, 3] * 40, [200, 17, 130] * 40),
    # several items for every SM of at most 32 sequences, in order of their keys: equal ones, rows without keys
    ("f16", 64, 32, 8, 16, [700, 1, 0, 500, 37, 130, 260], [700, 900, 10, 333, 1500, 129, 0]),
    ("bf16", 128, 56, 8, 32, [200, 90, 1, 36, 301, 37, 5, 250, 18], [1500, 90, 700, 36, 301, 2000, 5, 251, 18]),
    ("f16", 128, 300, 2, 16, [40, 3, 60], [50, 3, 900]),
    ("bf16", 64, 64, 8, 16, [33] * 32, [600] * 32),
    # single tokens: splits joined by a cluster, of which sequences use all, some, one or none
    ("bf16", 128, 32, 8, 64, [1, 2, 0, 1], [1000, 129, 70, 1]),
    ("f16", 64, 16, 16, 16, [1, 1, 1, 4], [700, 0, 300, 4]),
    # more splits than a cluster has: joined by groups of threads, a few and many
    ("f16", 64, 8, 8, 16, [1], [20000]),
    ("bf16", 128, 24, 2, 16, [1, 1], [11000, 900]),
    ("f16", 64, 32, 8, 32, [1, 2] * 20, [3000, 70, 900, 2, 1500, 17, 640, 2048, 1, 63] * 4),
]


def types():
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.mark.parametrize("case", SHAPES, ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}x{c[3]}-p{c[4]}-{c[5][:3]}-{c[6][:3]}")
@pytest.mark.parametrize("head_major", [False, True])
def test_attention(pkg, lib, case, head_major):
    import torch
    kind, d, heads, kvh, page, news, lens = case
    dt = types()[kind]
    pool = Pool(pkg, dt, kvh, d, page, lens, seed=d + heads + len(lens), head_major=head_major)
    pool.fill(lens)
    rows = sum(news)
    # strided rows, two padding rows behind the last sequence
    q = torch.randn((rows + 2, heads * d + 24), device="cuda").to(dt)[:, :heads * d]
    out = torch.full((rows + 2, heads * d + 8), 7.0, dtype=dt, device="cuda")
    attend(pkg, lib, pool, q, heads, news, lens, out[:, :heads * d])
    check_attention(pool, q, heads, news, lens, out[:, :heads * d])
    assert bool((out[rows:] == 7.0).all()) and bool((out[:, heads * d:] == 7.0).all())


@pytest.mark.parametrize("news,lens", [([1, 1], [500, 90]), ([150], [500])])
def test_attention_fp32_output_and_bounds_of_lengths(pkg, lib, news, lens):
    """An fp32 result; max_kv only splits the work, max_q may be larger than any chunk."""
    import torch
    pool = Pool(pkg, torch.float16, 8, 64, 16, lens, seed=3)
    pool.fill(lens)
    q = torch.randn((sum(news), 32 * 64), device="cuda").half()
    first = None
    for max_q, max_kv in [(None, None), (4096, 1), (None, 1 << 20), (max(news), 0)]:
        out = torch.zeros((sum(news), 32 * 64), device="cuda")
        attend(pkg, lib, pool, q, 32, news, lens, out, max_q=max_q, max_kv=max_kv)
        check_attention(pool, q, 32, news, lens, out)
        again = torch.zeros_like(out)
        attend(pkg, lib, pool, q, 32, news, lens, again, max_q=max_q, max_kv=max_kv)
        assert torch.equal(out, again)  # the same call, the same bits


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("news", [[1, 1], [140, 3]])
def test_attention_leaves_out_bad_pages(pkg, lib, page, news):
    """Page ids outside the pool (negative, past its end) hold no keys; a length past the table is cut."""
    import torch
    lens = [4 * page + 3, 3 * page]
    pool = Pool(pkg, torch.bfloat16, 2, 128, page, lens, seed=11)
    pool.fill(lens)
    pool.table[0, 1] = -1
    pool.table[0, 3] = pool.total
    pool.table[1, :3] = 2 ** 30  # the second sequence has no page at all: zeros
    dead = {0: torch.cat([torch.arange(page, 2 * page), torch.arange(3 * page, 4 * page)]).cuda(),
            1: torch.arange(0, 3 * page).cuda()}
    q = torch.randn((sum(news), 8 * 128), device="cuda").bfloat16()
    out = torch.full((sum(news), 8 * 128), 3.0, device="cuda").bfloat16()
    attend(pkg, lib, pool, q, 8, news, lens, out)

    class Seen:  # what remains readable: the dead keys' rows as zeros
        d, kv_heads, dtype = pool.d, pool.kv_heads, pool.dtype

        @staticmethod
        def rows(s, n):
            k = torch.zeros((n, 2, 128), dtype=torch.float64, device="cuda")
            v = torch.zeros_like(k)
            live = torch.ones(n, dtype=torch.bool, device="cuda")
            live[dead[s]] = False
            pos = live.nonzero()[:, 0]
            if len(pos):
                pg, sl = pool.where(s, pos)
                k[pos], v[pos] = pool.k[pg, sl].double(), pool.v[pg, sl].double()
            return k, v

    check_attention(Seen, q, 8, news, lens, out, dead=dead)
    assert bool((out[news[0]:] == 0).all())


@pytest.mark.parametrize("news", [[1], [96]])
def test_attention_large_scores(pkg, lib, news):
    """Scores that rise and fall by hundreds along the keys: the running maximum is rescaled, and
    sums neither overflow nor vanish."""
    import torch
    lens = [1500]
    pool = Pool(pkg, torch.float16, 4, 64, 16, lens, seed=5)
    pool.fill(lens)
    pg, sl = pool.where(0, torch.arange(1500, device="cuda"))
    ramp = torch.linspace(-30, 30, 1500, device="cuda") + 12 * torch.sin(torch.arange(1500, device="cuda") / 40.0)
    pool.k[pg, sl, :, 0] = ramp.half()[:, None]
    q = torch.randn((news[0], 16 * 64), device="cuda").half()
    q.view(news[0], 16, 64)[:, ::2, 0] = 60.0   # scores up to +-240, rising
    q.view(news[0], 16, 64)[:, 1::2, 0] = -60.0  # falling: the first keys win
    out = torch.zeros((news[0], 16 * 64), device="cuda").half()
    attend(pkg, lib, pool, q, 16, news, lens, out)
    check_attention(pool, q, 16, news, lens, out)


@pytest.mark.parametrize("news", [[1, 1, 1], [40, 1, 200]])
def test_attention_captured_and_replayed(pkg, lib, news):
    """One captured call, replayed over new lengths, tables and queries; another stream's eager call
    between the replays does not disturb it."""
    import torch
    cap = [900, 400, 700]
    pool = Pool(pkg, torch.float16, 8, 64, 16, cap, seed=8)
    pool.fill(cap)
    heads, rows = 32, sum(news)
    q = torch.randn((rows, heads * 64), device="cuda").half()
    out = torch.zeros((rows, heads * 64), device="cuda").half()
    lens = [300, 40, 250]
    cu = torch.tensor(np.cumsum([0] + news), dtype=torch.int32, device="cuda")
    kvl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    size = lib.llama_paged_attention_workspace(ctypes.byref(pool.desc), heads, rows, max(news), max(cap))
    ws = torch.empty((size + 16,), dtype=torch.uint8, device="cuda")

    def call(stream):
        rc = lib.llama_paged_attention(ctypes.byref(pool.desc), q.data_ptr(), q.stride(0), heads, cu.data_ptr(),
                                       kvl.data_ptr(), rows, max(news), max(cap), 0.125, out.data_ptr(), pkg.F16,
                                       out.stride(0), ws.data_ptr(), size, stream)
        assert rc == 0

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call(side.cuda_stream)
    for lens in ([300, 250, 250], cap, [40, 1, 200]):
        kvl.copy_(torch.tensor(lens, dtype=torch.int32))
        q.copy_(torch.randn_like(q))
        out.zero_()
        other = torch.zeros_like(out)
        graph.replay()
        attend(pkg, lib, pool, q, heads, news, lens, other)
        torch.cuda.synchronize()
        check_attention(pool, q, heads, news, lens, out, scale=0.125)
        check_attention(pool, q, heads, news, lens, other)


def test_attention_offsets_past_32_bits(pkg, lib):
    """Pages more than 2^31 elements into the pool."""
    import torch
    pages, page, kvh, d = 70_000, 256, 1, 128  # 2.3e9 elements each
    k = torch.empty((pages, page, kvh, d), dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    for news, lens in (([1], [300]), ([70], [300])):
        ids = torch.tensor([[69_999, 69_998]], dtype=torch.int32, device="cuda")
        k[69_998:].normal_()
        v[69_998:].normal_()
        pool = Pool(pkg, torch.bfloat16, kvh, d, page, lens, seed=1)
        pool.k, pool.v, pool.table, pool.total = k, v, ids, pages
        pool.desc.k, pool.desc.v, pool.desc.table = k.data_ptr(), v.data_ptr(), ids.data_ptr()
        pool.desc.num_pages, pool.desc.table_stride, pool.desc.table_width = pages, 2, 2
        pool.desc.page_stride, pool.desc.row_stride, pool.desc.head_stride = k.stride(0), k.stride(1), k.stride(2)
        q = torch.randn((news[0], 8 * d), device="cuda").bfloat16()
        out = torch.zeros_like(q)
        attend(pkg, lib, pool, q, 8, news, lens, out)
        check_attention(pool, q, 8, news, lens, out)


@pytest.mark.parametrize("news", [[1, 1, 1, 2], [40, 1, 130, 5]])
def test_sequences_by_slot(pkg, lib, news):
    """slots names each sequence's row of the table: any order, one row twice, one outside the table
    (no keys: zeros).  Append and attention agree on it."""
    import torch
    cap = [300, 200, 260]
    pool = Pool(pkg, torch.float16, 4, 64, 32, cap, seed=21)
    pool.fill(cap)
    heads, rows = 16, sum(news)
    slots = torch.tensor([2, 0, 2, 7], dtype=torch.int32, device="cuda")
    pool.desc.slots, pool.desc.table_rows, pool.desc.seqs = slots.data_ptr(), 3, 4
    lens = [250, 300, 190, 50]
    q = torch.randn((rows, heads * 64), device="cuda").half()
    out = torch.full((rows, heads * 64), 3.0, device="cuda").half()
    attend(pkg, lib, pool, q, heads, news, lens, out)

    class BySlot:
        d, kv_heads, dtype = pool.d, pool.kv_heads, pool.dtype

        @staticmethod
        def rows(s, n):
            return pool.rows([2, 0, 2][s], n)

    live = rows - news[3]
    check_attention(BySlot, q, heads, news[:3], lens[:3], out)
    assert bool((out[live:] == 0).all())
    # append of one row per sequence at its length
    cos, sin = rope(64, 512)
    qkv = torch.randn((4, (heads + 8) * 64), device="cuda")
    pos = torch.tensor([10, 20, 31, 5], dtype=torch.int32, device="cuda")
    seq = torch.arange(4, dtype=torch.int32, device="cuda")
    k0, v0 = pool.k.clone(), pool.v.clone()
    qo = torch.zeros((4, heads * 64), device="cuda").half()
    assert lib.llama_paged_append(ctypes.byref(pool.desc), qkv.data_ptr(), pkg.F32, qkv.stride(0), 4, heads, pos.data_ptr(),
                                  seq.data_ptr(), cos.data_ptr(), sin.data_ptr(), 512, qo.data_ptr(), pkg.F16,
                                  qo.stride(0), 0) == 0
    for i, (slot, p) in enumerate([(2, 10), (0, 20), (2, 31)]):
        pg, sl = pool.where(slot, torch.tensor([p], device="cuda"))
        assert torch.equal(pool.v[pg, sl].flatten(), qkv[i, (heads + 4) * 64:].half())
        k0[pg, sl], v0[pg, sl] = pool.k[pg, sl], pool.v[pg, sl]
    assert torch.equal(k0.nan_to_num(9.0), pool.k.nan_to_num(9.0)) and torch.equal(v0.nan_to_num(9.0), pool.v.nan_to_num(9.0))


def test_attention_workspace_is_checked(pkg, lib):
    import torch
    pool = Pool(pkg, torch.float16, 2, 64, 16, [5000], seed=2)
    pool.fill([5000])
    q = torch.randn((1, 8 * 64), device="cuda").half()
    out = torch.zeros_like(q)
    cu = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    kvl = torch.tensor([5000], dtype=torch.int32, device="cuda")
    size = lib.llama_paged_attention_workspace(ctypes.byref(pool.desc), 8, 1, 1, 5000)
    ws = torch.empty((size + 16,), dtype=torch.uint8, device="cuda")
    args = lambda p, n: (ctypes.byref(pool.desc), q.data_ptr(), q.stride(0), 8, cu.data_ptr(), kvl.data_ptr(), 1, 1, 5000,  # noqa: E731
                         0.125, out.data_ptr(), pkg.F16, out.stride(0), p, n, 0)
    assert lib.llama_paged_attention(*args(ws.data_ptr(), size)) == 0
    if size > 16:
        assert lib.llama_paged_attention(*args(ws.data_ptr(), size - 1)) == -2
        assert lib.llama_paged_attention(*args(None, size)) == -2
        assert lib.llama_paged_attention(*args(ws.data_ptr() + 8, size)) == -2
    host = torch.zeros((1, 8 * 64), dtype=torch.float16)
    bad = list(args(ws.data_ptr(), size))
    bad[10] = host.data_ptr()
    assert lib.llama_paged_attention(*bad) == -1
    torch.cuda.synchronize()


# ---- append ------------------------------------------------------------------------------------
def rope(d, n):
    import torch
    ang = torch.arange(n, dtype=torch.float64)[:, None] * (500000.0 ** (-torch.arange(d // 2) * 2.0 / d))[None, :]
    return torch.cos(ang).float().cuda(), torch.sin(ang).float().cuda()


@pytest.mark.parametrize("kind,in_kind,q_kind", [("f16", "f32", "f16"), ("f16", "f32", "f32"), ("f16", "f16", "f16"),
                                                 ("bf16", "f32", "bf16"), ("bf16", "f32", "f32"),
                                                 ("bf16", "bf16", "bf16")])
@pytest.mark.parametrize("d,heads,kvh,page", [(64, 32, 8, 16), (128, 7, 7, 64), (128, 6, 1, 256)])
def test_append(pkg, lib, kind, in_kind, q_kind, d, heads, kvh, page):
    import torch
    dt, it, qt = types()[kind], types()[in_kind], types()[q_kind]
    lens = [1, 40, 3 * page + 1, 700]
    news = [1, 40, 5, 1]
    pool = Pool(pkg, dt, kvh, d, page, lens, seed=4, head_major=d == 128, layers=3, layer=1)
    rows = sum(news) + 4
    n_pos = 4096
    cos, sin = rope(d, n_pos)
    qkv = torch.randn((rows, (heads + 2 * kvh) * d + 16), device="cuda").to(it)[:, :(heads + 2 * kvh) * d]
    pos = sum([list(range(n - m, n)) for m, n in zip(news, lens)], [])
    seq = sum([[i] * m for i, m in enumerate(news)], [])
    # padding rows: no sequence, a sequence past the table, positions outside the RoPE table
    pos, seq = pos + [3, 3, -1, n_pos], seq + [-1, 4, 1, 1]
    order = np.random.default_rng(0).permutation(rows)
    post = torch.tensor(np.array(pos)[order], dtype=torch.int32, device="cuda")
    seqt = torch.tensor(np.array(seq)[order], dtype=torch.int32, device="cuda")
    q = torch.full((rows, heads * d + 8), 5.0, dtype=qt, device="cuda")
    k0, v0 = pool.k.clone(), pool.v.clone()
    rc = lib.llama_paged_append(ctypes.byref(pool.desc), qkv.data_ptr(), codes(pkg)[it], qkv.stride(0), rows, heads,
                                post.data_ptr(), seqt.data_ptr(), cos.data_ptr(), sin.data_ptr(), n_pos, q.data_ptr(),
                                codes(pkg)[qt], q.stride(0), 0)
    assert rc == 0, lib.llama_engine_last_error(None)
    live = torch.tensor((order < rows - 4).nonzero()[0], device="cuda")
    idle = torch.tensor((order >= rows - 4).nonzero()[0], device="cuda")
    x = qkv[live].double().view(len(live), heads + 2 * kvh, d)
    p, s = post[live].long(), seqt[live].long()
    c, sn = cos[p].double()[:, None], sin[p].double()[:, None]
    a, b = x[:, :heads + kvh, :d // 2], x[:, :heads + kvh, d // 2:]
    ref = torch.cat([a * c - b * sn, a * sn + b * c], dim=2)
    mag = torch.cat([(a * c).abs() + (b * sn).abs(), (a * sn).abs() + (b * c).abs()], dim=2)

    def near(got, want, size, t):
        tol = 2.0 ** -23 * size + torch.finfo(t).eps / 2 * want.abs() + (2.0 ** -25 if t == torch.float16 else 0)
        assert bool(((got.double() - want).abs() <= tol).all())

    near(q[live, :heads * d].view(len(live), heads, d), ref[:, :heads], mag[:, :heads], qt)
    assert bool((q[idle] == 5.0).all()) and bool((q[:, heads * d:] == 5.0).all())
    pg, sl = pool.table[s, p // page].long(), p % page
    near(pool.k[pg, sl], ref[:, heads:], mag[:, heads:], dt)
    assert torch.equal(pool.v[pg, sl], x[:, heads + kvh:].to(dt))
    # nothing else was written
    k0[pg, sl], v0[pg, sl] = pool.k[pg, sl], pool.v[pg, sl]
    assert torch.equal(k0.nan_to_num(9.0), pool.k.nan_to_num(9.0))
    assert torch.equal(v0.nan_to_num(9.0), pool.v.nan_to_num(9.0))


def test_append_skips_bad_pages(pkg, lib):
    import torch
    pool = Pool(pkg, torch.float16, 2, 64, 16, [64, 64], seed=6)
    pool.table[0, 1] = -1
    pool.table[0, 2] = pool.total
    cos, sin = rope(64, 256)
    pos = torch.tensor([20, 40, 200, 3], dtype=torch.int32, device="cuda")  # two bad pages, past the table, good
    seq = torch.zeros(4, dtype=torch.int32, device="cuda")
    qkv = torch.randn((4, 8 * 64), device="cuda").half()
    q = torch.zeros((4, 4 * 64), device="cuda").half()
    assert lib.llama_paged_append(ctypes.byref(pool.desc), qkv.data_ptr(), pkg.F16, qkv.stride(0), 4, 4, pos.data_ptr(),
                                  seq.data_ptr(), cos.data_ptr(), sin.data_ptr(), 256, q.data_ptr(), pkg.F16,
                                  q.stride(0), 0) == 0
    written = (~torch.isnan(pool.k)).flatten(1).any(1).nonzero()[:, 0].tolist()
    assert written == [int(pool.table[0, 0])]
    assert int((~torch.isnan(pool.k)).sum()) == 2 * 64 and int((~torch.isnan(pool.v)).sum()) == 2 * 64
    assert bool((q != 0).any(dim=1).all())  # the queries are rotated all the same


def test_append_then_attend_step_by_step(pkg, lib):
    """A prompt appended and attended in chunks and single tokens gives the rows of one pass."""
    import torch
    heads, kvh, d, page, total = 8, 2, 64, 16, 150
    dt = torch.float16
    cos, sin = rope(d, 512)
    qkv = torch.randn((total, (heads + 2 * kvh) * d), device="cuda")
    outs = []
    for cuts in ([total], [1, 70, 1, 1, 64, 13], [37] + [1] * 20 + [93]):
        pool = Pool(pkg, dt, kvh, d, page, [total], seed=9)
        rows = []
        at = 0
        for n in cuts:
            q = torch.zeros((n, heads * d), dtype=dt, device="cuda")
            pos = torch.arange(at, at + n, dtype=torch.int32, device="cuda")
            seq = torch.zeros(n, dtype=torch.int32, device="cuda")
            part = qkv[at:at + n]
            assert lib.llama_paged_append(ctypes.byref(pool.desc), part.data_ptr(), pkg.F32, part.stride(0), n, heads,
                                          pos.data_ptr(), seq.data_ptr(), cos.data_ptr(), sin.data_ptr(), 512,
                                          q.data_ptr(), pkg.F16, q.stride(0), 0) == 0
            out = torch.zeros_like(q)
            attend(pkg, lib, pool, q, heads, [n], [at + n], out)
            check_attention(pool, q, heads, [n], [at + n], out)
            rows.append(out)
            at += n
        outs.append(torch.cat(rows))
    # different splits round the weights differently: each is within its bound of the same exact value
    for o in outs[1:]:
        assert float((o.double() - outs[0].double()).abs().max()) <= 4 * 2.0 ** -11 * 4.5


def test_calls_on_a_side_stream_are_ordered(pkg, lib):
    """The calls run on the stream they are given, behind that stream's earlier work."""
    import torch
    pool = Pool(pkg, torch.float16, 8, 64, 16, [600], seed=12)
    pool.fill([600])
    s = torch.cuda.Stream()
    q = torch.randn((1, 32 * 64), device="cuda").half()
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
        q.mul_(0.5)  # queued behind the sleep
        keep = attend(pkg, lib, pool, q, 32, [1], [600], out, stream=s.cuda_stream)
    s.synchronize()
    del keep
    check_attention(pool, q, 32, [1], [600], out)


@pytest.mark.parametrize("news", [[1, 2], [90, 3]])
@pytest.mark.parametrize("scale", [0.0, 1e-6, 0.6, -0.125])
def test_attention_scales(pkg, lib, news, scale):
    """A scale of zero is the mean of the keys' values, a negative one attends with -q."""
    import torch
    lens = [700, 150]
    pool = Pool(pkg, torch.bfloat16, 2, 128, 32, lens, seed=31)
    pool.fill(lens)
    q = torch.randn((sum(news), 8 * 128), device="cuda").bfloat16()
    out = torch.zeros_like(q)
    attend(pkg, lib, pool, q, 8, news, lens, out, scale=scale)
    check_attention(pool, -q if scale < 0 else q, 8, news, lens, out, scale=abs(scale))


def test_calls_at_once(pkg, lib):
    """Calls on several streams, each with its workspace, give the bits that they give alone."""
    import torch
    shapes = [(64, 32, 8, [1] * 20, [100 * i + 7 for i in range(20)]), (128, 28, 4, [200, 1, 330, 1], [900, 3000, 330, 40]),
              (64, 8, 8, [1], [9000]), (128, 16, 2, [150], [1200])]
    jobs, alone = [], []
    for i, (d, heads, kvh, news, lens) in enumerate(shapes):
        pool = Pool(pkg, torch.float16, kvh, d, 16, lens, seed=40 + i)
        pool.fill(lens)
        q = torch.randn((sum(news), heads * d), device="cuda").half()
        out = torch.zeros_like(q)
        attend(pkg, lib, pool, q, heads, news, lens, out)
        check_attention(pool, q, heads, news, lens, out)
        alone.append(out)
        cu = torch.tensor(np.cumsum([0] + news), dtype=torch.int32, device="cuda")
        kvl = torch.tensor(lens, dtype=torch.int32, device="cuda")
        size = lib.llama_paged_attention_workspace(ctypes.byref(pool.desc), heads, len(q), max(news), max(lens))
        ws = torch.empty((size + 16,), dtype=torch.uint8, device="cuda")
        jobs.append((pool, q, heads, news, lens, cu, kvl, size, ws, torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = [[torch.zeros_like(j[1]) for j in jobs] for _ in range(6)]
    torch.cuda.synchronize()
    for row in outs:
        for (pool, q, heads, news, lens, cu, kvl, size, ws, s), out in zip(jobs, row):
            rc = lib.llama_paged_attention(ctypes.byref(pool.desc), q.data_ptr(), q.stride(0), heads, cu.data_ptr(),
                                           kvl.data_ptr(), len(q), max(news), max(lens), pool.d ** -0.5, out.data_ptr(),
                                           pkg.F16, out.stride(0), ws.data_ptr(), size, s.cuda_stream)
            assert rc == 0
    torch.cuda.synchronize()
    for row in outs:
        for out, want in zip(row, alone):
            assert torch.equal(out, want)


@pytest.mark.parametrize("kvh,news,lens,bad", [
    (2, [200], [500], [402, 440, 480]), (8, [1], [700], [650]), (2, [20], [9000], [8995]), (8, [1], [20000], [19000])])
@pytest.mark.parametrize("kind,d", [("f16", 64), ("bf16", 128)])
def test_attention_of_a_nan_key(pkg, lib, kind, d, kvh, news, lens, bad):
    """A NaN among the keys that a row sees makes the row NaN, wherever the key lies in its tile (as the
    formula has it); rows that do not see it are as without it."""
    import torch
    dt = types()[kind]
    heads, n, kv = 4 * kvh, news[0], lens[0]
    for first in range(bad[0], bad[0] + 8 if n == 200 else bad[0] + 4):
        pool = Pool(pkg, dt, kvh, d, 16, lens, seed=50)
        pool.fill(lens)
        for j in [first] + bad[1:]:
            pg, sl = pool.where(0, torch.tensor([j], device="cuda"))
            pool.k[pg, sl, :, 3] = math.nan
        q = torch.randn((n, heads * d), device="cuda").to(dt)
        out = torch.zeros_like(q)
        attend(pkg, lib, pool, q, heads, news, lens, out)
        clear = max(0, first - (kv - n))  # rows whose position lies before the first bad key
        assert bool(out[clear:].isnan().all()), (first, out[clear:].isnan().float().mean().item())
        if clear:
            check_attention(pool, q, heads, [clear], [kv - n + clear], out)


@pytest.mark.parametrize("news", [[1, 2], [90, 3]])
def test_attention_at_the_ends_of_the_scale(pkg, lib, news):
    """The largest scales on equal scores, and a scale of zero on scores of 1e32: both are the mean."""
    import torch
    lens = [700, 150]
    for scale, size in ((3.0e38, 0.0), (-3.0e38, 0.0), (0.0, 1e15)):
        pool = Pool(pkg, torch.bfloat16, 2, 128, 32, lens, seed=33)
        pool.fill(lens)
        pg, sl = pool.where(0, torch.arange(700, device="cuda"))
        pool.k[pg, sl] *= size
        pg, sl = pool.where(1, torch.arange(150, device="cuda"))
        pool.k[pg, sl] *= size
        q = (torch.randn((sum(news), 8 * 128), device="cuda") * size).bfloat16()
        out = torch.zeros_like(q)
        attend(pkg, lib, pool, q, 8, news, lens, out, scale=scale)
        check_attention(pool, q, 8, news, lens, out, scale=0.0)


FIRST_CALLS = """
import ctypes, sys
sys.path[:0] = [{root!r}, {tests!r}]
import torch
from conftest import load_package
pkg = load_package()
from test_gpu_paged import Pool, rope
lib = pkg.LlamaEngineBindings().lib
news, lens, heads, kvh, d = [200, 1, 40, 1], [2600, 9000, 40, 700], 32, 8, 64
rows, vocab = sum(news), 4099
pool = Pool(pkg, torch.float16, kvh, d, 16, lens, seed=3)
pool.fill(lens)
i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
pos = i32(sum([list(range(n - m, n)) for m, n in zip(news, lens)], []))
seq = i32(sum([[i] * m for i, m in enumerate(news)], []))
cu, kvl = i32([0] + [sum(news[:i + 1]) for i in range(4)]), i32(lens)
cos, sin = rope(d, 9000)
qkv = torch.randn((rows, (heads + 2 * kvh) * d), device="cuda")
lg, u = torch.randn((5, vocab), device="cuda"), torch.rand(5, device="cuda")
k, p = i32([0, 5, 50, 0, 1]), torch.tensor([0.9, 1.0, 0.8, 1.0, 1.0], device="cuda")
size = lib.llama_paged_attention_workspace(ctypes.byref(pool.desc), heads, rows, 200, 9000)
ws = torch.empty((size + 16,), dtype=torch.uint8, device="cuda")
q, out = [torch.zeros((rows, heads * d), dtype=torch.float16, device="cuda") for _ in range(2)]
ids = torch.zeros(5, dtype=torch.int32, device="cuda")
def calls(s):
    rc = lib.llama_paged_append(ctypes.byref(pool.desc), qkv.data_ptr(), pkg.F32, qkv.stride(0), rows, heads, pos.data_ptr(),
                                seq.data_ptr(), cos.data_ptr(), sin.data_ptr(), 9000, q.data_ptr(), pkg.F16, q.stride(0), s)
    assert rc == 0, lib.llama_engine_last_error(None)
    rc = lib.llama_paged_attention(ctypes.byref(pool.desc), q.data_ptr(), q.stride(0), heads, cu.data_ptr(), kvl.data_ptr(),
                                   rows, 200, 9000, 0.125, out.data_ptr(), pkg.F16, out.stride(0), ws.data_ptr(), size, s)
    assert rc == 0, lib.llama_engine_last_error(None)
    rc = lib.llama_sample_rows(lg.data_ptr(), pkg.F32, vocab, 5, vocab, None, k.data_ptr(), p.data_ptr(), None, u.data_ptr(),
                               ids.data_ptr(), s)
    assert rc == 0, lib.llama_engine_last_error(None)
torch.cuda.synchronize()
side = torch.cuda.Stream()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=side):
    calls(side.cuda_stream)
graph.replay()
torch.cuda.synchronize()
first = [x.clone() for x in (q, out, ids, pool.k.nan_to_num(9.0), pool.v.nan_to_num(9.0))]
for x in (q, out, ids):
    x.zero_()
calls(0)
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(first, (q, out, ids, pool.k.nan_to_num(9.0), pool.v.nan_to_num(9.0))))
assert bool((out != 0).any(dim=1).all())
print("same")
"""


def test_the_first_calls_of_a_process_may_be_captured(pkg, gpu_available):
    """Nothing has to run before a capture: the captured calls replay to the bits of later eager ones."""
    import subprocess
    import sys
    from conftest import ROOT
    code = FIRST_CALLS.format(root=str(ROOT), tests=str(ROOT / "tests"))
    res = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and res.stdout.strip() == "same", res.stderr[-2000:]
