"""Engines with a paged KV cache (llama_engine_create_paged) and batched sampling
(llama_engine_sample_batch).

A paged engine runs the flat engine's batched steps on other attention operators, so its logits
differ by the rounding of q, k, v and the softmax's weights to the cache's type: each moves a layer's
attention output by about h = eps / 2 of its size (four roundings, and k's and q's again through the
scores), and two layers pass that on.  16 h of the largest logit is the bound used: 7.8e-3 for fp16,
6.3e-2 for bf16.
"""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_sample import oracle

pytestmark = pytest.mark.gpu
H = {1: 2.0 ** -11, 2: 2.0 ** -8}


@pytest.fixture(scope="module")
def bindings(pkg, gpu_available):
    return pkg.LlamaEngineBindings()


def near(got, ref, cache_type):
    return float(np.abs(got - ref).max()) <= 16 * H[cache_type] * float(np.abs(ref).max())


@pytest.mark.parametrize("cache_type,page", [(1, 16), (2, 64), (1, 256)])
def test_prefill_decode_and_scores_match_the_flat_engine(pkg, bindings, small_model, cache_type, page):
    flat = pkg.LlamaEngine(str(small_model), bindings, device=0, max_batch=4, max_seq_len=512)
    eng = pkg.LlamaEngine(str(small_model), bindings, device=0, max_batch=4, max_seq_len=512,
                          num_pages=4 * 512 // page, page_size=page, cache_type=cache_type)
    rng = np.random.default_rng(3)
    ids = [int(t) for t in rng.integers(0, 4096, 300)]
    try:
        assert eng.batch_path == "tensor-core"
        for e in (flat, eng):
            e.prefill(ids[:250], 0, True)
        assert near(eng.get_logits(), flat.get_logits(), cache_type)
        for i in range(250, 262):  # single tokens
            for e in (flat, eng):
                e.forward_token(ids[i], i, True)
            assert near(eng.get_logits(), flat.get_logits(), cache_type)
            assert eng.sample(0.0) == int(np.argmax(eng.get_logits()))
        for e in (flat, eng):  # a further chunk over the cache
            e.prefill(ids[262:], 262, True)
        assert near(eng.get_logits(), flat.get_logits(), cache_type)
        got = eng.generate_greedy(ids[0], 300, 5)
        tok, pos = ids[0], 300
        for want in got:  # the loop's ids are the greedy ids of its own steps
            eng.forward_token(tok, pos, True)
            assert int(np.argmax(eng.get_logits())) == want
            tok, pos = want, pos + 1
        lp_f, _ = flat.score_tokens(ids[:120], 0)
        lp_p, _ = eng.score_tokens(ids[:120], 0)
        assert float(np.abs(lp_f - lp_p).max()) <= 2 * 16 * H[cache_type] * float(np.abs(flat.get_logits()).max())
        assert eng.free_pages == eng.max_batch * 512 // page - (305 + page - 1) // page
    finally:
        flat.close()
        eng.close()


def test_positions_that_were_skipped_within_a_page(pkg, bindings, small_model):
    """Rows of a fresh page that are never fed count as keys of zeros, as in the flat engine."""
    flat = pkg.LlamaEngine(str(small_model), bindings, device=0, max_batch=1, max_seq_len=64)
    eng = pkg.LlamaEngine(str(small_model), bindings, device=0, max_batch=1, max_seq_len=64, num_pages=2, page_size=32)
    try:
        for e in (flat, eng):
            e.forward_token(77, 20, True)
        assert near(eng.get_logits(), flat.get_logits(), 1)
        assert eng.free_pages == 1
    finally:
        flat.close()
        eng.close()


def test_batched_rows_of_many_slots(pkg, bindings, small_model):
    """Rows in any order: single positions, several positions of a slot in one call, slots interleaved."""
    flat = pkg.LlamaEngine(str(small_model), bindings, device=0, max_batch=8, max_seq_len=256)
    eng = pkg.LlamaEngine(str(small_model), bindings, device=0, max_batch=8, max_seq_len=256, num_pages=8 * 16,
                          page_size=16)
    rng = np.random.default_rng(5)
    try:
        # prompts of different lengths for five slots in one call without logits (40 + 3 + 17 + 1 + 70 rows)
        rows = [(s, p) for s, n in ((6, 40), (0, 3), (3, 17), (7, 1), (2, 70)) for p in range(n)]
        tok = [int(t) for t in rng.integers(0, 4096, len(rows))]
        for e in (flat, eng):
            e.forward_batch(tok, [p for _, p in rows], [s for s, _ in rows], compute_logits=False)
        nxt = {6: 40, 0: 3, 3: 17, 7: 1, 2: 70}
        for step in range(4):
            order = [[2, 0, 7, 3, 6], [0, 2, 3, 6, 7], [6, 0, 6, 2, 0, 3], [7, 2, 2, 2, 3]][step]
            rows = []
            for s in order:
                rows.append((s, nxt[s]))
                nxt[s] += 1
            tok = [int(t) for t in rng.integers(0, 4096, len(rows))]
            for e in (flat, eng):
                e.forward_batch(tok, [p for _, p in rows], [s for s, _ in rows])
            for i in range(len(rows)):
                assert near(eng.get_logits_batch(i), flat.get_logits_batch(i), 1), (step, i)
            assert eng.argmax_batch(len(rows)) == [int(np.argmax(eng.get_logits_batch(i))) for i in range(len(rows))]
    finally:
        flat.close()
        eng.close()


def test_pages_run_out_and_come_back(pkg, bindings, small_model):
    eng = pkg.LlamaEngine(str(small_model), bindings, device=0, max_batch=3, max_seq_len=256, num_pages=6, page_size=16)
    try:
        assert eng.free_pages == 6
        eng.forward_batch(list(range(20, 60)), list(range(40)), [0] * 40, compute_logits=False)  # 3 pages
        eng.forward_batch([1], [0], [1])
        ref = eng.get_logits_batch(0)
        assert eng.free_pages == 2
        with pytest.raises(RuntimeError, match="out of KV cache pages"):
            eng.forward_batch(list(range(40)), list(range(40)), [2] * 40, compute_logits=False)
        with pytest.raises(RuntimeError, match="out of KV cache pages"):
            eng.prefill(list(range(100)), 40, False)
        assert eng.free_pages == 2  # nothing was taken by the refused calls
        eng.release_slot(0)
        assert eng.free_pages == 5
        eng.forward_batch(list(range(40)), list(range(40)), [2] * 40, compute_logits=False)
        assert eng.free_pages == 2
        eng.forward_batch([1], [0], [1])  # slot 1 kept its own page
        assert np.array_equal(eng.get_logits_batch(0), ref)
        with pytest.raises(RuntimeError):
            eng.release_slot(3)
        # a new sequence in the released slot, on pages that others used before
        eng.release_slot(2)
        eng.prefill([5, 6, 7, 8], 0, True)
        again = eng.get_logits()
        eng.release_slot(0)
        eng.prefill([5, 6, 7, 8], 0, True)
        assert np.array_equal(eng.get_logits(), again)
    finally:
        eng.close()


def test_flat_engines_refuse_page_calls(pkg, bindings, small_model):
    eng = pkg.LlamaEngine(str(small_model), bindings, device=0, max_batch=2, max_seq_len=64)
    try:
        assert eng.free_pages == -1
        with pytest.raises(RuntimeError, match="paged"):
            eng.release_slot(0)
    finally:
        eng.close()


@pytest.mark.parametrize("paged", [False, True])
def test_sample_batch(pkg, bindings, small_model, paged):
    """Ids by the sampler's definition over the logits that get_logits_batch returns."""
    extra = dict(num_pages=64, page_size=16) if paged else {}
    eng = pkg.LlamaEngine(str(small_model), bindings, device=0, max_batch=6, max_seq_len=64, **extra)
    rng = np.random.default_rng(7)
    try:
        for step in range(3):
            n = 6 - step
            eng.forward_batch([int(t) for t in rng.integers(0, 4096, n)], [step] * n, list(range(n)))
            t = np.float32(rng.choice([0.0, 0.7, 1.0, 2.0], n))
            k = np.int32(rng.choice([0, 5, 100], n))
            p = np.float32(rng.choice([1.0, 0.9, 0.4], n))
            m = np.float32(rng.choice([0.0, 0.05], n))
            u = np.float32(rng.random(n))
            rows = [eng.get_logits_batch(i).astype(np.float64) for i in range(n)]
            ids = eng.sample_batch(u, temperature=t, top_k=k, top_p=p, min_p=m)
            assert ids == [oracle(rows[i], float(t[i]), int(k[i]), float(p[i]), float(m[i]), float(u[i])) for i in range(n)]
            assert eng.sample_batch(u, temperature=0.0) == eng.argmax_batch(n)
            assert eng.sample_batch(u) == [oracle(rows[i], 1.0, 0, 1.0, 0.0, float(u[i])) for i in range(n)]
            assert np.array_equal(eng.get_logits_batch(n - 1), rows[n - 1].astype(np.float32))  # unchanged
        with pytest.raises(RuntimeError, match="max_batch"):
            eng.sample_batch(np.zeros(7))
    finally:
        eng.close()


def test_serving_loop_of_the_three_operators(pkg, bindings, small_model):
    """Prompts of three slots, then sampled steps: append, attention and sampling as a server runs them.
    The same numbers give the same ids again on released and reused pages."""
    eng = pkg.LlamaEngine(str(small_model), bindings, device=0, max_batch=3, max_seq_len=128, num_pages=18, page_size=16)
    prompts = [[11, 523, 77, 3000, 42], list(range(100, 133)), [9]]
    runs = []
    try:
        for _ in range(2):
            rng = np.random.default_rng(1)
            for s, ids in enumerate(prompts):
                if len(ids) > 1:
                    eng.forward_batch(ids[:-1], list(range(len(ids) - 1)), [s] * (len(ids) - 1), compute_logits=False)
            last, pos, out = [p[-1] for p in prompts], [len(p) - 1 for p in prompts], []
            for _ in range(12):
                eng.forward_batch(last, pos, [0, 1, 2])
                last = eng.sample_batch(rng.random(3), temperature=[0.8, 1.0, 0.0], top_k=[40, 0, 0], top_p=[0.95, 0.9, 1.0])
                pos = [p + 1 for p in pos]
                out.append(last)
            runs.append(out)
            for s in (2, 0, 1):
                eng.release_slot(s)
            assert eng.free_pages == 18
        assert runs[0] == runs[1]
    finally:
        eng.close()


def test_a_wait_that_runs_out_is_reported(pkg, bindings, small_model):
    """The chunk attention's product issuer waits on a phase that nothing completes (1 ms bound): the
    step drains, the next waiting call fails with the reason, and the engine works again."""
    eng = pkg.LlamaEngine(str(small_model), bindings, device=0, max_batch=2, max_seq_len=128, num_pages=16, page_size=16)
    lib = bindings.lib
    ids = list(range(50, 90))
    try:
        eng.prefill(ids, 0, True)
        ref = eng.get_logits()
        assert lib.llama_engine_debug_waits(eng.handle, 1_000_000, 20) == 0
        eng.prefill(ids, 0, True)
        with pytest.raises(RuntimeError):
            eng.get_logits()
        assert "paged attention" in bindings.last_error(eng.handle)
        assert lib.llama_engine_debug_waits(eng.handle, 0, 0) == 0
        eng.prefill(ids, 0, True)
        assert np.array_equal(eng.get_logits(), ref)
    finally:
        eng.close()


def test_create_refusals(pkg, bindings, small_model, chain_model):
    lib = bindings.lib
    for pages, size, kind in ((0, 16, 1), (4, 8, 1), (4, 48, 1), (4, 512, 1), (4, 16, 0), (4, 16, 3)):
        assert not lib.llama_engine_create_paged(str(small_model).encode(), 0, 1, 64, pages, size, kind)
        assert b"create_paged" in lib.llama_engine_last_error(None)
    # a geometry without the tensor-core batched path
    assert not lib.llama_engine_create_paged(str(chain_model).encode(), 0, 1, 64, 4, 16, 1)
    assert b"batched path" in lib.llama_engine_last_error(None)


def test_steps_are_captured_after_many_prompt_shapes(pkg, bindings, small_model):
    """Prompts of ever new lengths take no decode step's graph: a decode shape that comes after them is
    replayed from its first step on, a prompt's shape from its second.  Replays give the same bits."""
    eng = pkg.LlamaEngine(str(small_model), bindings, device=0, max_batch=2, max_seq_len=128, num_pages=16, page_size=16)
    try:
        before = eng.graph_steps
        for n in range(2, 82):
            eng.forward_batch(list(range(n)), list(range(n)), [0] * n, compute_logits=False)
            eng.release_slot(0)
        assert eng.graph_steps == before
        eng.prefill(list(range(20)), 0, False)
        seen = []
        for i in range(3):  # the same decode step again and again
            eng.forward_batch([7, 9], [20, 0], [0, 1])
            assert eng.graph_steps == before + i + 1
            seen.append(np.stack([eng.get_logits_batch(r) for r in range(2)]))
        assert all(np.array_equal(seen[0], x) for x in seen[1:])
        before = eng.graph_steps
        seen = []
        for i in range(3):  # a prompt with a single token beside it: launched, then captured, then replayed
            eng.forward_batch([7, 9, 11], [20, 0, 1], [0, 1, 1], compute_logits=False)
            eng.forward_batch([7, 9], [21, 2], [0, 1])
            assert eng.graph_steps == before + i + (i + 1)
            seen.append(np.stack([eng.get_logits_batch(r) for r in range(2)]))
        assert all(np.array_equal(seen[0], x) for x in seen[1:])
    finally:
        eng.close()


@pytest.mark.parametrize("paged", [False, True])
def test_more_step_shapes_than_graphs(pkg, bindings, small_model, paged):
    """A shape beyond the graphs that are held takes the place of the one used the longest ago once it has
    come four times; results do not depend on which steps are replayed."""
    extra = dict(num_pages=70, page_size=16) if paged else {}
    eng = pkg.LlamaEngine(str(small_model), bindings, device=0, max_batch=70, max_seq_len=16, **extra)
    try:
        def step(n):
            g = eng.graph_steps
            eng.forward_batch(list(range(n)), [0] * n, list(range(n)))
            return eng.graph_steps - g, eng.get_logits_batch(n - 1)

        first = [step(n) for n in range(1, 71)]
        assert [f[0] for f in first] == [1] * 64 + [0] * 6
        for want in (0, 0, 1, 1):  # the last shape's second to fifth steps
            got, logits = step(70)
            assert got == want and np.array_equal(logits, first[69][1])
        assert step(64)[0] == 1 and step(2)[0] == 1  # still held
        got, logits = step(1)  # gave its place
        assert got == 0 and np.array_equal(logits, first[0][1])
    finally:
        eng.close()


def test_operators_after_a_create_that_ran_out_of_memory(pkg, bindings, small_model):
    """An engine that could not be made leaves nothing behind that a later call would report as its own."""
    import torch
    lib = bindings.lib
    lg = torch.randn((3, 1000), device="cuda")
    u = torch.rand(3, device="cuda")
    ids = torch.full((3,), -5, dtype=torch.int32, device="cuda")
    for _ in range(2):
        assert not lib.llama_engine_create_paged(str(small_model).encode(), 0, 1, 64, 2 ** 31 - 1, 256, 1)
        assert b"out of memory" in lib.llama_engine_last_error(None)
        assert lib.llama_sample_rows(lg.data_ptr(), pkg.F32, 1000, 3, 1000, None, None, None, None, u.data_ptr(),
                                     ids.data_ptr(), 0) == 0, lib.llama_engine_last_error(None)
    assert not lib.llama_engine_create_paged(str(small_model).encode(), 0, 1, 64, 2 ** 31 - 1, 256, 1)
    eng = pkg.LlamaEngine(str(small_model), bindings, device=0, max_batch=1, max_seq_len=64, num_pages=4, page_size=16)
    try:
        eng.forward_token(5, 0, True)
        assert eng.sample_batch([0.5], temperature=0.0) == [int(np.argmax(eng.get_logits_batch(0)))]
    finally:
        eng.close()


def test_a_sampled_row_whose_wait_runs_out_is_reported(pkg, bindings, small_model):
    """The sampler waits for a copy that never comes (1 ms bound): the call fails, no id is returned, and
    the engine works again."""
    eng = pkg.LlamaEngine(str(small_model), bindings, device=0, max_batch=3, max_seq_len=64)
    lib = bindings.lib
    try:
        eng.forward_batch([5, 6, 7], [0, 0, 0], [0, 1, 2])
        ref = eng.sample_batch([0.2, 0.5, 0.9], top_k=40)
        assert lib.llama_engine_debug_waits(eng.handle, 1_000_000, 21) == 0
        for rules in (dict(), dict(top_k=40), dict(top_p=0.9), dict(temperature=0.0)):
            with pytest.raises(RuntimeError, match="timed out"):
                eng.sample_batch([0.2, 0.5, 0.9], **rules)
        eng.forward_batch([5, 6, 7], [0, 0, 0], [0, 1, 2])  # the step's own waits are not cut
        with pytest.raises(RuntimeError, match="timed out"):
            eng.sample_batch([0.2, 0.5, 0.9], top_k=40)
        assert lib.llama_engine_debug_waits(eng.handle, 0, 0) == 0
        assert eng.sample_batch([0.2, 0.5, 0.9], top_k=40) == ref
    finally:
        eng.close()
