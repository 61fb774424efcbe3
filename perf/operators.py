"""Measured cases of the paged-cache and sampling operators, with their plain forms.

``run`` computes an operator in elementary torch operations, or, with ``own`` true, calls
``llama_paged_append``, ``llama_paged_attention`` or ``llama_sample_rows`` of the engine library.
"""
from __future__ import annotations

import ctypes
import math
import random

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_CODES = {"f32": 0, "f16": 1, "bf16": 2}
_SIZES = {"f32": 4, "f16": 2, "bf16": 2}
_ROPE_POSITIONS = 8192


# ---- cases ---------------------------------------------------------------------------------
def _append(name, **kw):
    c = dict(op="append", seqs=1, new=1, start=0, ragged=False, heads=32, kv_heads=8, head_dim=64, page=16,
             in_type="f32", type="f16", q_type="f16", mix=1)
    c.update(kw)
    return dict(c, name=name) if name else c


def _attention(name, **kw):
    c = dict(op="attention", seqs=1, new=1, decodes=0, ctx=512, ragged=False, heads=32, kv_heads=8, head_dim=64,
             page=16, type="f16", mix=1)
    c.update(kw)
    return dict(c, name=name) if name else c


def _sample(name, **kw):
    c = dict(op="sample", rows=1, vocab=128256, type="f32", rules="all")
    c.update(kw)
    return dict(c, name=name) if name else c


def listed():
    return [
        # the K / V rows of a batch-64 decode step of the 1B model (32 heads of 64, 8 kv heads), from
        # the fp32 q | k | v product
        _append("append_decode64", seqs=64, new=1, start=1500, ragged=True),
        # a 2048-token prefill chunk of the 1B model
        _append("append_chunk2048", seqs=1, new=2048, start=2048),
        # ragged chunks of several prompts in 16 bits, heads of 128, padded to the step's row count
        _append("append_ragged_d128", seqs=13, new=700, start=3000, ragged=True, head_dim=128, heads=28, kv_heads=4,
                page=32, in_type="bf16", type="bf16", q_type="bf16", mix=5),
        # one user's decode step at a short context: latency
        _attention("decode_1x700", ctx=700),
        # batch-64 decode of the 1B model, contexts up to 2048, an idle slot among them
        _attention("decode_64x2048", seqs=64, decodes=64, ctx=2048, ragged=True, mix=3),
        # a full serving batch with heads of 128 and long contexts: the cache's bandwidth
        _attention("decode_128x8192_d128", seqs=128, decodes=128, ctx=8192, ragged=True, head_dim=128, type="bf16",
                   page=64, mix=4),
        # prefill of eight 2048-token prompts at once (the benchmark's prefill set)
        _attention("prefill_8x2048", seqs=8, new=2048, ctx=2048),
        # the next 512 tokens of a long document over its 32k context
        _attention("chunk_512x32768_d128", new=512, ctx=32768, head_dim=128, type="bf16", page=32),
        # decode rows and prompt chunks in one step, seven query heads per kv head, odd lengths
        _attention("mixed_24_d128", seqs=24, decodes=16, new=611, ctx=3001, ragged=True, head_dim=128, heads=28,
                   kv_heads=4, type="bf16", mix=6),
        # one user's next token
        _sample("sample_1", rows=1),
        # a batch-64 step with every user's own rules, greedy ones among them
        _sample("sample_64", rows=64),
        # a full batch in 16 bits, an odd vocabulary, no truncation: the whole row decides
        _sample("sample_256_bf16", rows=256, vocab=50257, type="bf16", rules="temperature"),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "sample"])
    mix = rng.randrange(1 << 30)
    if op == "sample":
        return _sample(None, rows=_spread(rng, 1, 256), vocab=_spread(rng, 1000, 128256),
                       type=rng.choice(["f32", "f16", "bf16"]), rules=rng.choice(["all", "temperature"]))
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8])
    shape = dict(kv_heads=kv_heads, heads=kv_heads * group, head_dim=rng.choice([64, 128]),
                 page=rng.choice([16, 32, 64, 128]), mix=mix)
    kind = rng.choice(["f16", "bf16"])
    if op == "append":
        seqs = _spread(rng, 1, 64)
        in_type = rng.choice(["f32", kind])
        return _append(None, seqs=seqs, new=_spread(rng, 1, max(1, 2048 // seqs)), start=rng.randrange(0, 4096),
                       ragged=rng.random() < 0.7, in_type=in_type, type=kind, q_type=rng.choice([in_type, kind]), **shape)
    form = rng.choice(["decode", "decode", "chunk", "mixed"])
    if form == "decode":
        seqs = _spread(rng, 1, 128)
        return _attention(None, seqs=seqs, decodes=seqs, ctx=_spread(rng, 16, 4096), ragged=rng.random() < 0.7,
                          type=kind, **shape)
    if form == "chunk":
        new = _spread(rng, 2, 1024)
        return _attention(None, seqs=rng.choice([1, 1, 2, 3]), new=new, ctx=_spread(rng, new, 8192),
                          ragged=rng.random() < 0.5, type=kind, **shape)
    seqs = rng.randrange(3, 17)
    new = _spread(rng, 2, 300)
    return _attention(None, seqs=seqs, decodes=rng.randrange(1, seqs), new=new, ctx=_spread(rng, new, 4096),
                      ragged=True, type=kind, **shape)


# ---- inputs --------------------------------------------------------------------------------
def _lengths(case):
    """(new tokens, keys) of each sequence: of the case alone, the same for every seed."""
    rng = random.Random(case["mix"])
    out = []
    for i in range(case["seqs"]):
        last = i == case["seqs"] - 1
        exact_len = last or not case["ragged"]
        if case["op"] == "append":
            n = case["new"] if exact_len else rng.randint(1, case["new"])
            out.append((n, n + (case["start"] if exact_len else rng.randint(0, case["start"]))))
            continue
        n = 1 if i < case["decodes"] else case["new"] if exact_len else rng.randint(1, case["new"])
        kv = case["ctx"] if exact_len else rng.randint(n, case["ctx"])
        if case["ragged"] and case["seqs"] >= 4 and i == 1:
            n = 0  # a slot without work in this step
        out.append((n, kv))
    return out


def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _pool(case, gen, lens, fill):
    """Page pools [pages][page][kv_heads][head_dim] and a table of shuffled pages for each sequence."""
    page = case["page"]
    need = [(kv + page - 1) // page for _, kv in lens]
    total = sum(need)
    width = max(need)
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    ends = np.cumsum([0] + need)
    idx = np.full((len(lens), width), 0, np.int64)
    for i, w in enumerate(need):
        idx[i, :w] = np.arange(ends[i], ends[i] + w)
    table = order[torch.from_numpy(idx).cuda()].contiguous()
    shape = (total, page, case["kv_heads"], case["head_dim"])
    dt = _TYPES[case["type"]]
    if not fill:
        return torch.zeros(shape, dtype=dt, device="cuda"), torch.zeros(shape, dtype=dt, device="cuda"), table
    k = torch.empty(shape, dtype=dt, device="cuda")
    v = torch.empty(shape, dtype=dt, device="cuda")
    k.normal_(generator=gen)
    v.normal_(generator=gen)
    k[..., :4] += 1.5  # a few channels with an offset, as keys have
    return k, v, table


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    st = {"case": case}
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        lg = torch.randn((rows, vocab), generator=gen, device="cuda") * 2.5
        # 200 likely ids a row (distinct ones), their logits falling with the logarithm of the rank
        rank = torch.randperm(200, generator=gen, device="cuda")[None, :] + 1.0
        peaks = (torch.randint(0, vocab, (rows, 1), generator=gen, device="cuda")
                 + torch.arange(200, device="cuda")[None, :] * (vocab // 200)) % vocab
        lg.scatter_(1, peaks, (16.0 - 1.2 * torch.log(rank)).expand(rows, 200).contiguous())
        st["logits"] = lg.to(_TYPES[case["type"]])

        def pick(values, dtype):
            v = torch.tensor(values, dtype=dtype, device="cuda")
            return v[torch.randint(0, len(values), (rows,), generator=gen, device="cuda")].contiguous()

        every = case["rules"] == "all"
        st["temperature"] = pick([0.7, 0.8, 1.0, 1.2, 0.0] if every and rows > 1 else [0.7, 0.8, 1.0, 1.2], torch.float32)
        st["top_k"] = pick([50, 20, 200, 0, 1000] if every else [0], torch.int32)
        st["top_p"] = pick([0.9, 0.95, 0.8, 1.0] if every else [1.0], torch.float32)
        st["min_p"] = pick([0.0, 0.0, 0.05, 0.02] if every else [0.0], torch.float32)
        st["uniform"] = torch.rand((rows,), generator=gen, device="cuda")
        st["ids"] = torch.zeros((rows,), dtype=torch.int32, device="cuda")
    else:
        lens = _lengths(case)
        heads, kvh, d = case["heads"], case["kv_heads"], case["head_dim"]
        live = sum(n for n, _ in lens)
        st["lens"], st["live"] = lens, live
        st["k"], st["v"], st["table"] = _pool(case, gen, lens, case["op"] == "attention")
        if case["op"] == "append":
            rows = live + (5 if case["ragged"] else 0)  # a padded step: rows of no sequence at its end
            st["rows"] = rows
            st["qkv"] = _normal(gen, (rows, (heads + 2 * kvh) * d), _TYPES[case["in_type"]])
            pos = np.concatenate([np.arange(kv - n, kv) for n, kv in lens] + [np.zeros(rows - live)])
            seq = np.concatenate([np.full(n, i) for i, (n, _) in enumerate(lens)] + [np.full(rows - live, -1)])
            st["pos"] = torch.from_numpy(pos.astype(np.int32)).cuda()
            st["seq"] = torch.from_numpy(seq.astype(np.int32)).cuda()
            freq = 500000.0 ** (-np.arange(d // 2) * 2.0 / d)
            ang = np.arange(_ROPE_POSITIONS)[:, None] * freq[None, :]
            st["cos"] = torch.from_numpy(np.cos(ang).astype(np.float32)).cuda()
            st["sin"] = torch.from_numpy(np.sin(ang).astype(np.float32)).cuda()
            st["q"] = torch.zeros((rows, heads * d), dtype=_TYPES[case["q_type"]], device="cuda")
        else:
            dt = _TYPES[case["type"]]
            st["q"] = _normal(gen, (live, heads * d), dt)
            st["out"] = torch.zeros((live, heads * d), dtype=dt, device="cuda")
            st["max_q"] = max(n for n, _ in lens)
            st["max_kv"] = max(kv for _, kv in lens)
            st["cu_q"] = torch.from_numpy(np.cumsum([0] + [n for n, _ in lens]).astype(np.int32)).cuda()
            st["kv_len"] = torch.tensor([kv for _, kv in lens], dtype=torch.int32, device="cuda")
    if own:
        _bind(st)  # the library, the cache descriptor and the workspace that a program keeps
    return st


# ---- the framework's calls -----------------------------------------------------------------
_package = None


def _load():
    global _package
    if _package is None:
        import importlib.util
        import sys
        from pathlib import Path

        home = Path(__file__).resolve().parent.parent / "llama3-signed-4bit_b200"
        name = "llama3_signed_4bit_b200"
        if name not in sys.modules:
            spec = importlib.util.spec_from_file_location(name, home / "__init__.py", submodule_search_locations=[str(home)])
            mod = importlib.util.module_from_spec(spec)
            sys.modules[name] = mod
            spec.loader.exec_module(mod)
        pkg = sys.modules[name]
        _package = (pkg, pkg.LlamaEngineBindings().lib)
    return _package


def _bind(st):
    pkg, lib = _load()
    case = st["case"]
    st["lib"] = lib
    if case["op"] == "sample":
        return
    kv = pkg.PagedKV(k=st["k"].data_ptr(), v=st["v"].data_ptr(), type=_CODES[case["type"]], num_pages=st["k"].shape[0],
                     page_size=case["page"], kv_heads=case["kv_heads"], head_dim=case["head_dim"],
                     page_stride=st["k"].stride(0), row_stride=st["k"].stride(1), head_stride=st["k"].stride(2),
                     table=st["table"].data_ptr(), table_stride=st["table"].stride(0), table_width=st["table"].shape[1],
                     seqs=case["seqs"])
    st["kv"] = ctypes.byref(kv)
    if case["op"] == "attention":
        size = lib.llama_paged_attention_workspace(st["kv"], case["heads"], st["live"], st["max_q"], st["max_kv"])
        st["work"] = torch.empty((max(size, 16),), dtype=torch.uint8, device="cuda")


def _run_own(st):
    case = st["case"]
    lib = st["lib"]
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "append":
        rc = lib.llama_paged_append(st["kv"], st["qkv"].data_ptr(), _CODES[case["in_type"]], st["qkv"].stride(0), st["rows"],
                                    case["heads"], st["pos"].data_ptr(), st["seq"].data_ptr(), st["cos"].data_ptr(),
                                    st["sin"].data_ptr(), _ROPE_POSITIONS, st["q"].data_ptr(), _CODES[case["q_type"]],
                                    st["q"].stride(0), stream)
        out = [st["q"], st["k"], st["v"]]
    elif case["op"] == "attention":
        rc = lib.llama_paged_attention(st["kv"], st["q"].data_ptr(), st["q"].stride(0), case["heads"],
                                       st["cu_q"].data_ptr(), st["kv_len"].data_ptr(), st["live"], st["max_q"], st["max_kv"],
                                       1.0 / math.sqrt(case["head_dim"]), st["out"].data_ptr(), _CODES[case["type"]],
                                       st["out"].stride(0), st["work"].data_ptr(), st["work"].numel(), stream)
        out = st["out"]
    else:
        lg = st["logits"]
        rc = lib.llama_sample_rows(lg.data_ptr(), _CODES[case["type"]], lg.stride(0), case["rows"], case["vocab"],
                                   st["temperature"].data_ptr(), st["top_k"].data_ptr(), st["top_p"].data_ptr(),
                                   st["min_p"].data_ptr(), st["uniform"].data_ptr(), st["ids"].data_ptr(), stream)
        out = st["ids"]
    if rc != 0:
        raise RuntimeError(f"{case['op']} refused: {lib.llama_engine_last_error(None).decode()}")
    return out


# ---- plain forms ---------------------------------------------------------------------------
def _plain_append(st):
    case, live = st["case"], st["live"]
    heads, kvh, d = case["heads"], case["kv_heads"], case["head_dim"]
    x = st["qkv"][:live].float().view(live, heads + 2 * kvh, d)
    pos, seq = st["pos"][:live].long(), st["seq"][:live].long()
    c, s = st["cos"][pos][:, None, :], st["sin"][pos][:, None, :]
    a, b = x[:, :heads + kvh, :d // 2], x[:, :heads + kvh, d // 2:]
    r = torch.cat([a * c - b * s, a * s + b * c], dim=2)
    st["q"][:live] = r[:, :heads].reshape(live, heads * d).to(st["q"].dtype)
    page = st["table"][seq, pos // case["page"]].long()
    st["k"][page, pos % case["page"]] = r[:, heads:].to(st["k"].dtype)
    st["v"][page, pos % case["page"]] = x[:, heads + kvh:].to(st["v"].dtype)
    return [st["q"], st["k"], st["v"]]


def _plain_attention(st):
    """Every sequence padded to the longest: scores [seq][kv head][token, group][key]."""
    case = st["case"]
    heads, kvh, d = case["heads"], case["kv_heads"], case["head_dim"]
    g, nmax, kmax = heads // kvh, st["max_q"], st["max_kv"]
    seqs = case["seqs"]
    pages = st["table"].long()
    k = st["k"][pages].view(seqs, -1, kvh, d)[:, :kmax].permute(0, 2, 3, 1).float()
    v = st["v"][pages].view(seqs, -1, kvh, d)[:, :kmax].permute(0, 2, 1, 3).float()
    first, n, length = st["cu_q"][:-1].long(), st["cu_q"][1:].long() - st["cu_q"][:-1].long(), st["kv_len"].long()
    tok = torch.arange(nmax, device="cuda")
    row = (first[:, None] + tok[None, :]).clamp(max=st["live"] - 1)
    q = st["q"].view(st["live"], kvh, g, d)[row].float()                       # [seq][token][kv head][group][d]
    q = q.permute(0, 2, 1, 3, 4).reshape(seqs, kvh, nmax * g, d)
    s = torch.matmul(q, k) * (1.0 / math.sqrt(d))
    last = (length - n)[:, None] + tok[None, :]                                # position of each token
    seen = torch.arange(kmax, device="cuda")[None, None, :] <= last[:, :, None]
    seen = seen.repeat_interleave(g, dim=1)[:, None]
    s = s.masked_fill_(~seen, -math.inf)
    s = s.sub_(s.amax(dim=3, keepdim=True)).exp_()
    o = torch.matmul(s, v) / s.sum(dim=3, keepdim=True)
    o = o.view(seqs, kvh, nmax, g, d).permute(0, 2, 1, 3, 4).reshape(seqs * nmax, heads * d)
    # back to the packed rows: row t of sequence i is padded row i * nmax + t
    owner = torch.searchsorted(st["cu_q"], torch.arange(st["live"], device="cuda", dtype=torch.int32), right=True) - 1
    return o[owner * nmax + torch.arange(st["live"], device="cuda") - first[owner]].to(st["q"].dtype)


def _plain_sample(st):
    """Weights in 64 bits: a draw lands next to a border of two ids now and then."""
    rows, vocab = st["logits"].shape
    lg = st["logits"].double()
    order = torch.sort(lg, dim=1, descending=True, stable=True)
    top = order.values[:, :1]
    greedy = st["temperature"] <= 0.01
    t = torch.where(greedy, 1.0, st["temperature"]).double()[:, None]
    w = torch.exp((order.values - top) / t)
    cum = torch.cumsum(w, dim=1)
    rank = torch.arange(vocab, device="cuda")[None, :]
    k = torch.where(st["top_k"] > 0, st["top_k"].long(), vocab).clamp(max=vocab)[:, None]
    mass_k = torch.gather(cum, 1, k - 1)
    p = st["top_p"].double()[:, None]
    in_p = (p >= 1.0) | (cum - w < p * mass_k)
    kept = (rank < k) & in_p & (w >= st["min_p"].double()[:, None]) & (~greedy[:, None] | (rank == 0))
    by_index = torch.zeros_like(w).scatter_(1, order.indices, torch.where(kept, w, 0.0))
    run_mass = torch.cumsum(by_index, dim=1)
    goal = st["uniform"].double()[:, None] * run_mass[:, -1:]
    return (run_mass <= goal).sum(dim=1).clamp(max=vocab - 1).to(torch.int32)


def run(state):
    if own:
        return _run_own(state)
    return {"append": _plain_append, "attention": _plain_attention, "sample": _plain_sample}[state["case"]["op"]](state)


# ---- what a pass cannot do without ---------------------------------------------------------
def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * _SIZES[case["type"]] + case["rows"] * 24, "flops": 4 * n}
    lens = _lengths(case)
    live = sum(n for n, _ in lens)
    heads, kvh, d = case["heads"], case["kv_heads"], case["head_dim"]
    size = _SIZES[case["type"]]
    if case["op"] == "append":
        spots = len({p for n, kv in lens for p in range(kv - n, kv)})
        return {"bytes": live * ((heads + 2 * kvh) * d * _SIZES[case["in_type"]] + heads * d * _SIZES[case["q_type"]]
                                 + 2 * kvh * d * size + 8) + spots * d * 4,
                "flops": 3 * live * (heads + kvh) * d}
    seen = sum(n * (kv - n) + n * (n + 1) // 2 for n, kv in lens)
    keys = sum(kv for n, kv in lens if n > 0)
    return {"bytes": 2 * live * heads * d * size + 2 * keys * kvh * d * size, "flops": 4 * seen * heads * d}


# ---- the definition in 64 bits -------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "sample":
        ids = []
        names = ("logits", "temperature", "top_k", "top_p", "min_p", "uniform")
        columns = [st[n].double().cpu().numpy() for n in names]
        for lg, temp, k, p, m, u in zip(*columns):
            best = int(np.argmax(lg))
            if temp <= 0.01:
                ids.append(best)
                continue
            w = np.exp((lg - lg[best]) / temp)
            order = np.argsort(-lg, kind="stable")
            if k > 0:
                order = order[:int(k)]
            c = np.cumsum(w[order])
            if p < 1.0:
                order = order[:int(np.searchsorted(c, p * c[-1], side="left")) + 1]
            order = np.sort(order[w[order] >= m])
            c = np.cumsum(w[order])
            ids.append(int(order[min(int(np.searchsorted(c, u * c[-1], side="right")), len(order) - 1)]))
        return torch.tensor(ids, dtype=torch.int32)
    heads, kvh, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    table = st["table"].cpu().numpy()
    if case["op"] == "append":
        q, k, v = st["q"].double(), st["k"].double(), st["v"].double()
        x = st["qkv"].double().reshape(-1, heads + 2 * kvh, d // 2 * 2)
        at = 0
        for i, (n, kv) in enumerate(st["lens"]):
            where = np.arange(kv - n, kv)
            turn = torch.complex(st["cos"][kv - n:kv].double(), st["sin"][kv - n:kv].double())[:, None, :]
            part = x[at:at + n, :heads + kvh]
            z = torch.complex(part[..., :d // 2], part[..., d // 2:]) * turn
            flat = torch.cat([z.real, z.imag], dim=-1)
            q[at:at + n] = flat[:, :heads].reshape(n, heads * d)
            pg = torch.from_numpy(table[i][where // page].astype(np.int64)).cuda()
            sl = torch.from_numpy(where % page).cuda()
            k[pg, sl] = flat[:, heads:]
            v[pg, sl] = x[at:at + n, heads + kvh:]
            at += n
        return [q, k, v]
    if work(case)["flops"] > 4e11:
        return None
    out = torch.zeros((st["live"], heads, d), dtype=torch.float64, device="cuda")
    g = heads // kvh
    at = 0
    for i, (n, kv) in enumerate(st["lens"]):
        if n == 0:
            continue
        pg = torch.from_numpy(table[i][:(kv + page - 1) // page].astype(np.int64)).cuda()
        kk = st["k"][pg].reshape(-1, kvh, d)[:kv].double()
        vv = st["v"][pg].reshape(-1, kvh, d)[:kv].double()
        qq = st["q"][at:at + n].double().view(n, heads, d)
        hide = torch.ones((n, kv), dtype=torch.bool, device="cuda").triu(kv - n + 1)
        for h in range(kvh):
            e = torch.einsum("tgd,kd->gtk", qq[:, h * g:(h + 1) * g], kk[:, h]) / math.sqrt(d)
            p = torch.exp(e - e.masked_fill(hide, -math.inf).amax(dim=-1, keepdim=True)) * ~hide
            out[at:at + n, h * g:(h + 1) * g] = torch.einsum("gtk,kd->tgd", p / p.sum(dim=-1, keepdim=True), vv[:, h])
        at += n
    return out.view(st["live"], heads * d)
