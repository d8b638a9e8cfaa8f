"""The page table's side of evictions, and a cache whose eviction fails (no GPU)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from klcquant_amd import ops
from klcquant_amd.attention import AttentionConfig
from klcquant_amd.paged_kv import BatchedAttention, PagedKVCache, PageTable


def cut(table, seqs, keep):
    plan = table.eviction(seqs, keep)
    table.evict(plan, keep)
    return plan


def consistent(table):
    """Every page is free or held by as many sequences as the table says."""
    holders = np.zeros(table.n_pages, int)
    for s in np.flatnonzero(table._lengths >= 0):
        np.add.at(holders, table.pages(int(s)), 1)
    assert (holders == table._holders).all()
    assert sorted(table._free) == np.flatnonzero(holders == 0).tolist()


def test_a_cut_frees_pages_and_keeps_positions():
    t = PageTable(20, 16)
    a, b = t.add(), t.add()
    t.extend([a, b], [100, 30])
    before = t.pages(a)
    plan = cut(t, [a, b], 40)
    assert plan["seqs"].tolist() == [a] and plan["keys"].tolist() == [100] and plan["src"] == [] and plan["pages"][0].tolist() == before
    assert t.length(a) == 40 and t.pages(a) == before[:3] and t.length(b) == 30
    consistent(t)
    x = t.extend([a, b], [10, 1])
    assert x["positions"].tolist() == list(range(100, 110)) + [30]
    assert x["slots"].tolist()[:8] == [before[2] * 16 + i for i in range(8, 16)]
    assert x["keys"].tolist() == [50, 31] and x["lengths"].tolist() == list(range(41, 51)) + [31]
    t.undo_extend([a, b], [10, 1])
    assert t.length(a) == 40 and t.extend([a])["positions"].tolist() == [100]
    child, = t.fork(a)[0]
    assert t.extend([child])["positions"].tolist() == [101]
    t.free(a)
    assert t.add() == a and t.extend([a])["positions"].tolist() == [0]
    consistent(t)


def test_shared_pages_are_copied_unless_one_holds_them():
    t = PageTable(20, 16)
    a = t.add()
    t.extend([a], [64])
    b, c = t.fork(a, 2)[0]
    shared = t.pages(a)
    plan = cut(t, [a, b], 20)  # c keeps the four pages
    assert plan["src"] == shared[:2] * 2 and t.pages(c) == shared
    assert len({*t.pages(a), *t.pages(b), *shared}) == 8
    consistent(t)
    plan = cut(t, [c], 40)  # alone by now
    assert plan["src"] == [] and t.pages(c) == shared[:3]
    d, = t.fork(c)[0]
    plan = cut(t, [c, d], 33)  # the first of them gets copies, the other has the pages by then
    assert plan["src"] == shared[:2] and t.pages(d)[:2] == shared[:2]
    consistent(t)


def test_all_or_nothing():
    t = PageTable(6, 16)
    a = t.add()
    t.extend([a], [64])
    b, = t.fork(a)[0]
    state = (t._free[:], t._holders.tolist(), t.pages(a), t.pages(b))
    with pytest.raises(RuntimeError, match="taken"):
        t.eviction([a], 48)
    plan = t.eviction([a], 20)
    assert state == (t._free[:], t._holders.tolist(), t.pages(a), t.pages(b)) and len(plan["dst"]) == 2
    with pytest.raises(KeyError):
        t.eviction([7], 20)
    with pytest.raises(ValueError):
        t.eviction([a], 0)
    with pytest.raises(ValueError):
        t.eviction([a, a], 20)
    assert t.eviction([a, b], 64)["seqs"].size == 0
    consistent(t)


def test_a_compaction_after_a_cut():
    t = PageTable(20, 16)
    a, b = t.add(), t.add()
    t.extend([a, b], [100, 90])
    cut(t, [a], 20)
    src, dst = t.compact()
    assert max(t.pages(a) + t.pages(b)) == 7 and len(src) == len(dst)
    consistent(t)


def test_an_eviction_that_fails_leaves_the_cache(monkeypatch):
    cache = PagedKVCache("cpu", 2, 2, 64, 20, 16, "bf16", weighted=(4, 200))
    a = cache.add()
    cache.extend([a], [100])
    b, = cache.table.fork(a)[0]

    def state():
        return cache.table._free[:], cache.table._holders.tolist(), cache.table.pages(a), cache.table.pages(b), cache.length(a)

    def broken(*args, **kwargs):
        raise RuntimeError("no launch")

    before = state()
    for name in ("copy_pages", "evict_keys"):
        monkeypatch.setattr(ops, "copy_pages", lambda *x: None)
        monkeypatch.setattr(ops, name, broken)
        with pytest.raises(RuntimeError, match="no launch"):
            cache.evict([a, b], 40)
        assert state() == before
    calls = []
    monkeypatch.setattr(ops, "copy_pages", lambda pool, src, dst: calls.append((src, dst)))
    monkeypatch.setattr(ops, "evict_keys", lambda *x, **kw: calls.append((x[2].tolist(), x[3].tolist(), x[4].tolist(), x[5], kw)))
    assert cache.evict([a, b], 40, recent=10, first=2) == [a, b]
    tables, lengths, rows, keep, kw = calls[1]
    assert calls[0][0] == before[2][:3] and tables[0][:3] == calls[0][1] and tables[1] == before[3]
    assert (lengths, rows, keep, kw) == ([100, 100], [a, b], 40, dict(recent=10, first=2))
    assert cache.length(a) == cache.length(b) == 40
    consistent(cache.table)


def test_refusals():
    plain = PagedKVCache("cpu", 1, 2, 64, 20, 16)
    with pytest.raises(ValueError, match="without weights"):
        plain.evict([plain.add()], 10)
    for weighted in ((0, 5), (5, 0), (5,), (-1, 5)):
        with pytest.raises(ValueError, match="weights of"):
            PagedKVCache("cpu", 1, 2, 64, 20, 16, weighted=weighted)
    cache = PagedKVCache("cpu", 1, 2, 64, 20, 16, weighted=(2, 50))
    a = cache.add()
    for kw in (dict(keep=10, recent=-1), dict(keep=10, first=-1), dict(keep=10, recent=6, first=5), dict(keep=0), dict(keep=-3)):
        with pytest.raises(ValueError):
            cache.evict([a], **kw)
    with pytest.raises(TypeError):
        cache.evict([a], 10.5)
    with pytest.raises(RuntimeError, match="50 keys"):
        cache.extend([a], [51])
    assert cache.length(a) == 0 and cache.stats()["free_pages"] == 20
    cache.extend([a], [50])
    cache.add()
    for call in (cache.add, lambda: cache.fork(a)):
        with pytest.raises(RuntimeError, match="2 sequences"):
            call()
    assert cache.stats()["sequences"] == 2
    with pytest.raises(ValueError):
        BatchedAttention(AttentionConfig(512, 8, 2, 64), first_tokens=-1)
    with pytest.raises(ValueError, match="GPU"):
        ops.attention_plan([1], [1], 8, 2, 64, device="cpu")
    assert torch.equal(cache.weights, torch.zeros(1, 2, 2, 50))
