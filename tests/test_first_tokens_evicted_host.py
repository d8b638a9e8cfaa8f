"""First tokens beside windows and evictions that would put other keys in their places (no GPU)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from klcquant_amd import ops
from klcquant_amd.attention import AttentionConfig
from klcquant_amd.paged_kv import BatchedAttention, PagedKVCache, PageTable


def test_a_table_knows_how_many_are_in_place():
    t = PageTable(40, 16)
    a, b = t.add(), t.add()
    whole = t.extend([a, b], [100, 90])["firsts"].tolist()
    assert min(whole) > 90

    def cut(seqs, keep, first):
        t.evict(t.eviction(seqs, keep), keep, first)

    cut([a], 60, 8)
    assert t.extend([a, b])["firsts"].tolist() == [8, whole[1]]
    child, = t.fork(a)[0]
    cut([a, child], 50, 20)  # what was moved before stays moved
    assert t.extend([a, b, child])["firsts"].tolist() == [8, whole[1], 8]
    cut([a], 40, 3)
    assert t.extend([a, child])["firsts"].tolist() == [3, 8]
    cut([b], 200, 0)  # not cut
    assert t.extend([b])["firsts"].tolist() == whole[1:]
    t.free(a)
    assert t.add() == a and t.extend([a])["firsts"].tolist() == whole[:1]
    more = [t.add() for _ in range(9)]  # past the first eight
    assert t.extend(more)["firsts"].tolist() == whole[:1] * 9


def test_evictions_and_layers_that_do_not_go_together(monkeypatch):
    monkeypatch.setattr(ops, "evict_keys", lambda *x, **kw: None)
    config = AttentionConfig(256, 4, 2, 64)
    cache = PagedKVCache("cpu", 1, 2, 64, 40, 16, "bf16", weighted=(4, 200))
    a, b = cache.add(), cache.add()
    cache.extend([a, b], [100, 100])
    assert cache.evict([a], 50, 10, 4) == [a]
    batch, other = cache.extend([a, b]), cache.extend([b])
    hidden, tensors = torch.zeros(2, 256).bfloat16(), {}

    def run(first_tokens, batch, window):
        BatchedAttention(config, first_tokens).forward(0, hidden[:batch.tokens], tensors, batch, cache, window)

    with pytest.raises(ValueError, match="cut to the first 4"):
        run(5, batch, 32)
    assert cache.first_tokens == 0
    # these get as far as the layer's tensors, of which there are none
    for first_tokens, of, window in ((4, batch, 32), (5, batch, None), (5, batch, 0), (5, other, 32)):
        with pytest.raises(KeyError):
            run(first_tokens, of, window)
    assert cache.first_tokens == 5
    before = cache.length(b)
    with pytest.raises(ValueError, match="first 4 keys kept, of 5"):
        cache.evict([b], 50, 10, 4)
    assert cache.length(b) == before and cache.evict([b], 50, 10, 5) == [b]
    with pytest.raises(ValueError, match="first 3"):
        cache.evict([b], 3, 0, 3)
