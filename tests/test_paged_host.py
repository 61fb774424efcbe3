"""Refusals of the paged-cache and sampling operators: they need no GPU, since every argument is
checked before any device work."""
from __future__ import annotations

import ctypes

import pytest

PTR = 0x10000  # never dereferenced: the calls refuse first


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.LlamaEngineBindings().lib


def cache(pkg, **kw):
    a = dict(k=PTR, v=PTR, type=pkg.F16, num_pages=4, page_size=16, kv_heads=2, head_dim=64, page_stride=16 * 128,
             row_stride=128, head_stride=64, table=PTR, table_stride=4, table_width=4, seqs=3)
    a.update(kw)
    return pkg.PagedKV(**a)


def append(lib, kv, **kw):
    a = dict(qkv=PTR, type=0, ld=8 * 64, rows=5, heads=4, pos=PTR, seq=PTR, cos=PTR, sin=PTR, n_pos=100, q=PTR, q_type=1,
             q_ld=4 * 64)
    a.update(kw)
    return lib.llama_paged_append(ctypes.byref(kv) if kv else None, *a.values(), None)


def attend(lib, kv, **kw):
    a = dict(q=PTR, q_ld=4 * 64, heads=4, cu=PTR, kvl=PTR, rows=5, max_q=5, max_kv=60, scale=0.125, out=PTR, out_type=1,
             out_ld=4 * 64, ws=PTR, size=1 << 40)
    a.update(kw)
    return lib.llama_paged_attention(ctypes.byref(kv) if kv else None, *a.values(), None)


def sample(lib, **kw):
    a = dict(logits=PTR, type=0, ld=1000, rows=3, vocab=1000, t=None, k=None, p=None, m=None, u=PTR, out=PTR)
    a.update(kw)
    return lib.llama_sample_rows(*a.values(), None)


BAD_CACHES = [dict(k=None), dict(v=None), dict(table=None), dict(type=0), dict(type=3), dict(head_dim=96),
              dict(page_size=8), dict(page_size=24), dict(page_size=512), dict(num_pages=0), dict(kv_heads=0),
              dict(seqs=0), dict(table_width=0), dict(table_width=5), dict(k=PTR + 8), dict(v=PTR + 2),
              dict(row_stride=132), dict(head_stride=32), dict(page_stride=-128), dict(page_stride=1 << 40),
              dict(table_width=1 << 27, table_stride=1 << 27), dict(slots=PTR), dict(slots=PTR, table_rows=-1),
              dict(table_rows=3)]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
def test_bad_cache_is_refused(pkg, lib, bad):
    kv = cache(pkg, **bad)
    assert append(lib, kv) == -1
    assert attend(lib, kv) == -1
    assert b"llama_paged_attention" in lib.llama_engine_last_error(None)
    assert lib.llama_paged_attention_workspace(ctypes.byref(kv), 4, 5, 5, 60) == 0


@pytest.mark.parametrize("bad", [dict(qkv=None), dict(pos=None), dict(seq=None), dict(cos=None), dict(sin=None),
                                 dict(q=None), dict(type=2), dict(type=9), dict(q_type=2), dict(type=1, q_type=0),
                                 dict(rows=-1), dict(n_pos=0), dict(heads=0), dict(heads=3), dict(ld=8 * 64 - 4),
                                 dict(ld=8 * 64 + 2), dict(q_ld=4 * 64 - 8), dict(q_ld=4 * 64 + 4), dict(qkv=PTR + 4),
                                 dict(q=PTR + 8), dict(cos=PTR + 4)], ids=str)
def test_append_refusals(pkg, lib, bad):
    assert append(lib, cache(pkg), **bad) == -1
    assert append(lib, None) == -1


@pytest.mark.parametrize("bad", [dict(q=None), dict(cu=None), dict(kvl=None), dict(out=None), dict(out_type=2),
                                 dict(out_type=7), dict(rows=-1), dict(max_q=-1), dict(max_kv=-1), dict(heads=0),
                                 dict(heads=5), dict(heads=8192), dict(scale=float("nan")), dict(scale=float("inf")),
                                 dict(q_ld=4 * 64 - 8), dict(q_ld=4 * 64 + 4), dict(out_ld=4 * 64 - 8),
                                 dict(out_ld=4 * 64 + 4), dict(q=PTR + 8), dict(out=PTR + 8)], ids=str)
def test_attention_refusals(pkg, lib, bad):
    assert attend(lib, cache(pkg), **bad) == -1
    assert attend(lib, None) == -1


@pytest.mark.parametrize("bad,rc", [(dict(logits=None), -1), (dict(u=None), -1), (dict(out=None), -1), (dict(type=3), -1),
                                    (dict(rows=-1), -1), (dict(vocab=0), -1), (dict(ld=999), -1),
                                    (dict(logits=PTR + 1), -1), (dict(vocab=(1 << 18) + 1, ld=1 << 20), -2)], ids=str)
def test_sample_refusals(lib, bad, rc):
    assert sample(lib, **bad) == rc
    assert b"llama_sample_rows" in lib.llama_engine_last_error(None)


def test_no_rows_is_no_work(pkg, lib):
    kv = cache(pkg)
    assert append(lib, kv, rows=0) == 0
    assert attend(lib, kv, rows=0) == 0
    assert sample(lib, rows=0) == 0


def test_engine_entry_points_refuse_null(lib):
    assert not lib.llama_engine_create_paged(None, 0, 1, 64, 4, 16, 1)
    assert lib.llama_engine_release_slot(None, 0) == -1
    assert lib.llama_engine_free_pages(None) == -1
    assert lib.llama_engine_sample_batch(None, None, None, None, None, None, 1, None) == -1


def test_host_memory_is_refused(pkg, lib):
    """Pointers that are no device memory are refused, not read."""
    kv = cache(pkg)
    assert append(lib, kv) == -1
    assert attend(lib, kv) == -1
    assert sample(lib) == -1
    assert b"CUDA device" in lib.llama_engine_last_error(None)


def test_workspace_of_sequences_without_rows(pkg, lib):
    """Described sequences that may have no row bound the splits of those that have one: a single row among
    many needs room for 8192 tiles and a split for each sequence, or as much as if all had rows."""
    part = (128 + 8) * 4 * 16  # bytes of a decode tile's part, heads of 128
    for keys in (2048, 8192, 32768):
        for seqs in (1, 16, 64, 256, 1000):
            kv = cache(pkg, num_pages=4096, page_size=64, kv_heads=8, head_dim=128, page_stride=64 * 1024, row_stride=1024,
                       head_stride=128, table_stride=keys // 64, table_width=keys // 64, seqs=seqs)
            size = lib.llama_paged_attention_workspace(ctypes.byref(kv), 32, 1, 1, keys)
            # keys of a split grow as the root of the call's keys: at most the root's splits and one for each pair
            full = (seqs * 8 * keys) ** 0.5 / 0.9 + seqs * 8
            assert size <= max(8192 + seqs * 8, full) * part
