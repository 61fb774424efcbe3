"""llama_sample_rows against its definition: weights rounded to 2^-44 in 64 bits, exact integer
masses, so an id is either right or wrong (no tolerance)."""
from __future__ import annotations

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
ONE = 1 << 44


@pytest.fixture(scope="module")
def lib(pkg, gpu_available):
    return pkg.LlamaEngineBindings().lib


def oracle(logits, t, k, p, m, u):
    """One row, by the definition; logits a float64 array."""
    l = np.where(np.isnan(logits) | (logits <= np.float32(-1e30)), -np.inf, logits)
    top = l.max()
    if top == -np.inf:
        return 0
    first = int(np.argmax(l))
    if not t > np.float32(0.01):
        return first
    with np.errstate(invalid="ignore"):
        x = np.where(l == top, 0.0, (l - top) / t if top < np.inf else -np.inf)
    w = np.floor(np.exp(x) * ONE + 0.5)
    w = np.where(l == -np.inf, 0, w).astype(np.int64)
    order = np.argsort(-l, kind="stable")
    order = order[l[order] > -np.inf]
    if k > 0:
        order = order[:k]
    if p < 1.0:
        total = int(w[order].sum())
        need = min(max(math.ceil(float(p) * float(total)) if p > 0 else 1, 1), total)
        order = order[:int(np.searchsorted(np.cumsum(w[order]), need, side="left")) + 1]
    if m > 0:
        order = order[w[order] >= math.ceil(min(float(m), 1.0) * ONE)]
    kept = np.sort(order)
    cum = np.cumsum(w[kept])
    total = int(cum[-1])
    goal = min(int(min(float(u), 1.0) * float(total)) if u > 0 else 0, total - 1)
    return int(kept[int(np.searchsorted(cum, goal, side="right"))])


def run(pkg, lib, logits, t=None, k=None, p=None, m=None, u=None, vocab=None, stream=0):
    import torch
    code = {torch.float32: pkg.F32, torch.float16: pkg.F16, torch.bfloat16: pkg.BF16}[logits.dtype]
    rows = logits.shape[0]
    vocab = logits.shape[1] if vocab is None else vocab
    dev = lambda x, dt: None if x is None else torch.tensor(np.broadcast_to(np.asarray(x), (rows,)).copy(), dtype=dt, device="cuda")  # noqa: E731
    args = [dev(t, torch.float32), dev(k, torch.int32), dev(p, torch.float32), dev(m, torch.float32), dev(u, torch.float32)]
    out = torch.full((rows + 1,), -5, dtype=torch.int32, device="cuda")
    ptr = [None if a is None else a.data_ptr() for a in args]
    rc = lib.llama_sample_rows(logits.data_ptr(), code, logits.stride(0), rows, vocab, *ptr, out.data_ptr(), stream)
    assert rc == 0, lib.llama_engine_last_error(None)
    torch.cuda.synchronize()
    assert int(out[rows]) == -5
    host = logits[:, :vocab].double().cpu().numpy()
    col = lambda i, d: np.full(rows, d) if args[i] is None else args[i].double().cpu().numpy()  # noqa: E731
    want = [oracle(host[r], col(0, 1.0)[r], int(col(1, 0)[r]), col(2, 1.0)[r], col(3, 0.0)[r], col(4, 0.0)[r])
            for r in range(rows)]
    assert out[:rows].tolist() == want
    return want


def rand(rows, vocab, dtype, seed, scale=3.0):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn((rows, vocab), generator=g, device="cuda") * scale).to(dtype)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("vocab", [1, 2, 31, 64, 1000, 4097, 32003, 128256, 262144])
def test_mixed_rules(pkg, lib, dtype, vocab):
    """Every rule alone and together, every row its own; 16-bit logits hold many equal values."""
    import torch
    rng = np.random.default_rng(vocab)
    n = 24
    lg = rand(n, vocab, getattr(torch, dtype), seed=vocab)
    run(pkg, lib, lg, t=rng.choice([0.3, 0.7, 1.0, 1.7, 0.0, 50.0], n), k=rng.choice([0, 1, 2, 50, 1000, 300000], n),
        p=rng.choice([1.0, 0.9, 0.5, 0.999, 0.0], n), m=rng.choice([0.0, 0.05, 0.3, 1.0], n), u=rng.random(n))


@pytest.mark.parametrize("rules", [dict(), dict(k=40), dict(p=0.9), dict(m=0.02), dict(k=100, p=0.8),
                                   dict(k=3000, p=0.97, m=0.001), dict(t=0.6), dict(t=0.0), dict(p=0.0), dict(m=1.0),
                                   dict(k=1), dict(t=0.6, p=0.5, k=7)], ids=str)
def test_each_rule_over_the_uniform_range(pkg, lib, rules):
    """The same row with 64 numbers from 0 to the last below 1; parameters that are off may be NULL."""
    import torch
    lg = rand(1, 50257, torch.float32, seed=3).expand(64, -1).contiguous()
    u = np.concatenate([np.linspace(0, 1, 63, endpoint=False), [1 - 2.0 ** -24]])
    run(pkg, lib, lg, u=u, **rules)


def test_strided_rows_and_unaligned_starts(pkg, lib):
    import torch
    for dt in (torch.float32, torch.float16, torch.bfloat16):
        buf = rand(9, 5003, dt, seed=5)
        for lo, hi in ((0, 5003), (1, 5000), (3, 4099)):
            run(pkg, lib, buf[:, lo:hi], t=0.9, k=60, p=0.95, u=np.linspace(0, 0.99, 9))


def test_masked_rows(pkg, lib):
    """Masked logits in every form: -inf, the type's lowest value, NaN, all of a row, all but one."""
    import torch
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        lg = rand(8, 3001, dt, seed=7)
        lg[0] = -math.inf
        lg[1] = torch.finfo(dt).min  # masked in fp32 and bf16, a plain equal value in fp16
        lg[2] = math.nan
        lg[3, ::2] = -math.inf
        lg[4] = -math.inf
        lg[4, 2999] = -3.0
        lg[5, 100:] = math.nan
        lg[6, 17] = math.inf
        lg[6, 2000] = math.inf
        for rules in (dict(), dict(k=5), dict(p=0.6), dict(m=0.1), dict(k=2000, p=0.9, m=0.01), dict(t=0.0)):
            run(pkg, lib, lg, u=np.linspace(0.05, 0.95, 8), **rules)


def test_ties(pkg, lib):
    """Equal logits: the order is the index's, cut anywhere; -0 and +0 are equal."""
    import torch
    lg = torch.zeros((40, 7000), device="cuda")
    lg[:, ::3] = -0.0
    run(pkg, lib, lg, k=np.arange(1, 41) * 170, u=np.linspace(0, 0.999, 40))
    run(pkg, lib, lg, p=np.linspace(0.01, 1.0, 40), u=0.9999)
    lg = (torch.randint(0, 6, (40, 7000), device="cuda")).float()
    run(pkg, lib, lg, k=np.arange(1, 41) * 170, p=np.linspace(0.2, 1.0, 40), m=0.003, u=np.linspace(0, 0.999, 40))


def test_odd_parameters(pkg, lib):
    """Out-of-range and non-finite parameters have a defined meaning."""
    import torch
    lg = rand(10, 2000, torch.float32, seed=2)
    nan, inf = math.nan, math.inf
    run(pkg, lib, lg, t=[nan, inf, 1e-3, -1.0, 1e30, 1.0, 1.0, 1.0, 1.0, 1.0], k=[-3, 5, 0, 0, 0, 2 ** 31 - 1, 0, 0, 0, 0],
        p=[1, 1, 1, 1, 0.5, 2.0, -1.0, nan, inf, 1], m=[0, 0, 0, 0, 0, -1.0, 0, nan, 5.0, 1e-30],
        u=[0.5, 0.5, 0.5, 0.5, 0.5, 1.0, -2.0, nan, inf, 0.99999994])


def test_wide_range_of_logits(pkg, lib):
    """Logits whose weights vanish at 2^-44, and a flat row of the largest vocabulary."""
    import torch
    lg = rand(6, 30000, torch.float32, seed=1, scale=200.0)
    run(pkg, lib, lg, p=[1, 0.9, 0.5, 1, 1, 0.999], k=[0, 0, 0, 500, 20000, 20000], u=np.linspace(0, 0.99, 6))
    flat = torch.zeros((4, 262144), device="cuda")
    run(pkg, lib, flat, p=[1, 0.5, 1, 0.25], k=[0, 0, 99999, 200000], u=[0.123456, 0.9, 0.5, 0.999])


def test_rows_do_not_depend_on_each_other(pkg, lib):
    """A row's id is the same alone and in a batch, and from call to call; captured calls replay."""
    import torch
    n, vocab = 70, 20011
    lg = rand(n, vocab, torch.float32, seed=9)
    u = torch.rand(n, device="cuda")
    t = torch.full((n,), 0.8, device="cuda")
    p = torch.full((n,), 0.95, device="cuda")
    out = torch.zeros(n, dtype=torch.int32, device="cuda")

    def call(r0, rows, stream=0):
        assert lib.llama_sample_rows(lg[r0:].data_ptr(), pkg.F32, vocab, rows, vocab, t[r0:].data_ptr(), None,
                                     p[r0:].data_ptr(), None, u[r0:].data_ptr(), out[r0:].data_ptr(), stream) == 0

    call(0, n)
    batch = out.clone()
    out.zero_()
    for r in range(n):
        call(r, 1)
    assert torch.equal(out, batch)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call(0, n, side.cuda_stream)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, batch)
    u.copy_(torch.rand(n, device="cuda"))
    graph.replay()
    torch.cuda.synchronize()
    replayed = out.clone()
    call(0, n)
    assert torch.equal(out, replayed)


@pytest.mark.parametrize("rows,vocab", [(149, 3001), (321, 700), (1024, 257), (1025, 130), (40, 128256)])
def test_many_rows_of_mixed_rules(pkg, lib, rows, vocab):
    """More rows than run at once: every row is taken exactly once, whatever its rule."""
    import torch
    rng = np.random.default_rng(rows)
    pick = lambda *v: [v[i] for i in rng.integers(0, len(v), rows)]  # noqa: E731
    lg = rand(rows, vocab, torch.float32, seed=rows, scale=1.0)
    run(pkg, lib, lg, t=pick(0.0, 0.7, 1.2), k=pick(0, 0, 40, 3000), p=pick(1.0, 0.9, 0.97, 0.5), m=pick(0.0, 0.02),
        u=rng.random(rows))


@pytest.mark.parametrize("vocab", [3001, 50257])
@pytest.mark.parametrize("top", [2e9, 1e20, 3e38, -5e29])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_maxima_whose_spacing_exceeds_the_temperature(pkg, lib, dtype, top, vocab):
    """Row maxima so large that fp32's next lower value is many temperatures away: only equals of the
    maximum have weight, whatever the rules, and masked ids (and the slots behind the row) have none."""
    import torch
    dt = getattr(torch, dtype)
    rng = np.random.default_rng(vocab)
    n = 24
    lg = rand(n, vocab, dt, seed=vocab) if top > 0 else torch.full((n, vocab), -9e29, device="cuda").to(dt)
    lg[:, ::5] = -math.inf
    lg[:, 1::7] = math.nan
    lg[:, 2::9] = -2e30
    lg[:, [vocab // 3, vocab // 3 + 1, vocab - 1]] = top
    if dtype == "float32":
        lg[::2, 8] = float(np.nextafter(np.float32(top), np.float32(-np.inf)))
    u = np.linspace(0, 1 - 2.0 ** -24, n)
    for t in (0.02, 0.7, 1.0):
        run(pkg, lib, lg, t=t, u=u)
        run(pkg, lib, lg, t=t, u=u, p=0.9)
        run(pkg, lib, lg, t=t, u=u, k=rng.choice([0, 1, 2, 3, 40, 2500], n), p=rng.choice([1.0, 0.3, 0.7], n),
            m=rng.choice([0.0, 0.5], n))


@pytest.mark.parametrize("top", [2.0 ** 31, 3e38])
def test_maxima_with_a_few_spacings_to_the_temperature(pkg, lib, top):
    """The logits with weight lie within a few fp32 steps of the maximum; the many below them have none,
    not even together (the last random number below 1 falls on the last id with weight)."""
    import torch
    vocab = 200001
    step = float(np.float32(top)) - float(np.nextafter(np.float32(top), np.float32(-np.inf)))
    for factor in (0.014, 0.03, 0.04, 0.06, 0.3, 2.0):
        t = np.float32(step * factor)
        lg = torch.zeros((6, vocab), device="cuda")
        lg[:, 0] = top
        near = torch.tensor([np.float32(top - step * i) for i in range(1, 40)], device="cuda")
        lg[3:, 1:40] = near
        lg[4, 100:] = -math.inf
        for p in (1.0, 0.99999994, 0.5):
            run(pkg, lib, lg, t=t, p=p, u=[1 - 2.0 ** -24, 0.5, 0.0, 1 - 2.0 ** -24, 1 - 2.0 ** -24, 0.9])
