"""A PagedKVCache whose device work fails holds what it held before the call (no GPU)."""

from __future__ import annotations

import copy

import pytest
import torch

from klcquant_amd import ops, paged_kv
from klcquant_amd.paged_kv import PagedKVCache


def state(cache):
    """What the table says, and what it will hand out next."""
    t = cache.table
    live = [s for s in range(len(t._lengths)) if t._lengths[s] >= 0]
    return ([(s, t.length(s), t.pages(s)) for s in live], list(t._free), t._holders.tolist(), cache.stats())


@pytest.fixture
def cache():
    c = PagedKVCache("cpu", 2, 2, 64, 20, 16, "bf16")
    a, b = c.add(), c.add()
    c.extend([a, b], [40, 70])
    c.table.fork(b, 1)
    return c


def broken(*args, **kwargs):
    raise RuntimeError("no launch")


def test_a_fork_that_fails_leaves_the_cache(cache, monkeypatch):
    monkeypatch.setattr(ops, "copy_pages", broken)
    before = state(cache)
    for count in (1, 3):
        with pytest.raises(RuntimeError, match="no launch"):
            cache.fork(0, count)
        assert state(cache) == before
    moves = []
    monkeypatch.setattr(ops, "copy_pages", lambda pool, src, dst: moves.append((src, dst)))
    children = cache.fork(0, 2)
    src, dst = moves[0]
    assert src == [cache.table.pages(0)[2]] * 2 and dst == [cache.table.pages(c)[2] for c in children]
    assert cache.fork(0, 0) == [] and len(moves) == 1


def test_a_compaction_that_fails_leaves_the_cache(cache, monkeypatch):
    cache.free(0)
    monkeypatch.setattr(ops, "copy_pages", broken)
    before, table = state(cache), copy.deepcopy(cache.table)
    with pytest.raises(RuntimeError, match="no launch"):
        cache.compact()
    assert state(cache) == before
    moves = []
    monkeypatch.setattr(ops, "copy_pages", lambda pool, src, dst: moves.append((src, dst)))
    held = cache.compact()
    assert moves == [table.compact()] and held == 20 - cache.stats()["free_pages"]
    assert state(cache)[0] == [(s, table.length(s), table.pages(s)) for s, _, _ in before[0]]


def test_an_extension_that_fails_leaves_the_cache(cache, monkeypatch):
    """All or nothing also where there is no memory for the batch's arrays."""
    before, real = state(cache), torch.empty
    monkeypatch.setattr(paged_kv.torch, "empty", broken)
    for seqs, counts in (([0], 1), ([0, 1, 2], [30, 1, 9]), ([1], 10)):
        with pytest.raises(RuntimeError, match="no launch"):
            cache.extend(seqs, counts)
        assert state(cache) == before
    monkeypatch.setattr(paged_kv.torch, "empty", real)
    monkeypatch.setattr(paged_kv.np, "repeat", broken)  # the table's own arrays
    with pytest.raises(RuntimeError, match="no launch"):
        cache.table.extend([2, 0], [40, 7])
    assert state(cache) == before
    monkeypatch.undo()
    batch = cache.extend([0, 1, 2], [30, 1, 9])
    assert batch.tokens == 40 and [cache.length(s) for s in range(3)] == [70, 71, 79]
