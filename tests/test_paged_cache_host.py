"""PageTable's bookkeeping against a model that keeps every sequence's tokens, and what it refuses (no GPU)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from klcquant_amd.paged_kv import BatchedAttention, PagedKVCache, PageTable
from klcquant_amd.attention import AttentionConfig, rope_cos_sin


class Model:
    """Tokens by sequence, and what the slots of the pages hold."""

    def __init__(self, n_pages, page):
        self.table, self.page = PageTable(n_pages, page), page
        self.slots = np.zeros(n_pages * page, np.int64)
        self.tokens, self.next = {}, 1

    def move(self, src, dst):
        assert not set(dst) & set(src) and len(set(dst)) == len(dst)
        pages = self.slots.reshape(-1, self.page)
        pages[dst] = pages[src]

    def extend(self, seqs, counts):
        before = [len(self.tokens[s]) for s in seqs]
        x = self.table.extend(seqs, counts)
        assert x["fresh"] == (not any(before)) and all(v.dtype == np.int32 for k, v in x.items() if k != "fresh")
        new = np.arange(self.next, self.next + x["slots"].size)
        self.next += new.size
        held = {slot for s in self.tokens for slot in self.at(s, len(self.tokens[s]))}
        assert len(set(x["slots"])) == new.size and not held & set(x["slots"])
        self.slots[x["slots"]] = new
        assert x["starts"].tolist() == [0] + np.cumsum(counts).tolist()
        for i, s in enumerate(seqs):
            a, b = x["starts"][i:i + 2]
            assert x["positions"][a:b].tolist() == list(range(before[i], before[i] + counts[i]))
            self.tokens[s] = self.tokens[s] + new[a:b].tolist()
            for t in range(a, a if x["fresh"] else b):  # what batch attention reads for this token
                n, shared = x["lengths"][t], x["prefix"].size * self.page
                slots = [x["prefix"][j // self.page] * self.page + j % self.page for j in range(shared)]
                slots += [x["tables"][t][j // self.page] * self.page + j % self.page for j in range(n)]
                assert n >= 1 and self.slots[slots].tolist() == self.tokens[s][:before[i] + t - a + 1]
        return x

    def at(self, s, n):
        pages = self.table.pages(s)
        return [pages[i // self.page] * self.page + i % self.page for i in range(n)]

    def check(self):
        for s, tokens in self.tokens.items():
            assert self.table.length(s) == len(tokens) and self.slots[self.at(s, len(tokens))].tolist() == tokens
        held = {p for s in self.tokens for p in self.table.pages(s)}
        stats = self.table.stats()
        assert stats["free_pages"] == self.table.n_pages - len(held) and not held & set(self.table._free)
        assert stats["sequences"] == len(self.tokens) and stats["tokens"] == sum(map(len, self.tokens.values()))


@pytest.mark.parametrize("seed", range(4))
def test_sequences_keep_their_tokens(seed):
    rng = np.random.RandomState(seed)
    m = Model(60, 16)
    refused = 0
    for _ in range(150):
        live = list(m.tokens)
        act = rng.choice(["add", "extend", "extend", "extend", "fork", "free", "compact"])
        if act == "add" or not live:
            m.tokens[m.table.add()] = []
        elif act == "extend":
            seqs = rng.permutation(live)[:rng.randint(1, len(live) + 1)].tolist()
            counts = rng.randint(1, 40 if rng.rand() < 0.3 else 4, len(seqs)).tolist()
            try:
                m.extend(seqs, counts)
            except RuntimeError:
                refused += 1
                m.table.free(live[0])
                del m.tokens[live[0]]
        elif act == "fork" and len(live) < 14:
            parent = live[rng.randint(len(live))]
            try:
                children, src, dst = m.table.fork(parent, int(rng.randint(0, 4)))
            except RuntimeError:
                refused += 1
                continue
            m.move(src, dst)
            for c in children:
                assert c not in m.tokens
                m.tokens[c] = list(m.tokens[parent])
        elif act == "free":
            m.table.free(live[0])
            del m.tokens[live[0]]
        elif act == "compact":
            m.move(*m.table.compact())
            held = {p for s in m.tokens for p in m.table.pages(s)}
            assert held == set(range(len(held)))
        m.check()
    assert m.next > 500


def test_shared_pages_are_the_prefix():
    m = Model(40, 16)
    a = m.table.add()
    m.tokens[a] = []
    m.extend([a], [70])
    children, src, dst = m.table.fork(a, 3)
    assert len(src) == 3 and set(src) == {m.table.pages(a)[4]}
    m.move(src, dst)
    m.tokens.update({c: list(m.tokens[a]) for c in children})
    x = m.extend(children, [1, 1, 1])
    assert x["prefix"].tolist() == m.table.pages(a)[:4] and x["lengths"].tolist() == [7, 7, 7] and x["tables"].shape == (3, 1)
    b = m.table.add()
    m.tokens[b] = []
    assert m.extend([children[0], b], [1, 2])["prefix"].size == 0
    assert m.table.stats()["shared_pages"] == 4
    for s in (a, *children):
        m.table.free(s)
        del m.tokens[s]
    m.check()


def test_refusals():
    t = PageTable(4, 16)
    a, b = t.add(), t.add()
    for seqs, counts, error in (([a, a], 1, ValueError), ([7], 1, KeyError), ([-1], 1, KeyError), ([], 1, ValueError),
                                ([a], 0, ValueError), ([a], [1.5], ValueError), ([a, b], [1, 2, 3], ValueError),
                                ([a, b], [40, 17], RuntimeError), ([a], 1 << 30, ValueError)):
        with pytest.raises(error):
            t.extend(seqs, counts)
    assert t.stats()["free_pages"] == 4 and t.length(a) == t.length(b) == 0  # all or none
    t.extend([a], 50)
    with pytest.raises(RuntimeError, match="1 needed, 0 free"):
        t.fork(a)
    assert t.stats()["sequences"] == 2
    t.free(b)
    with pytest.raises(KeyError):
        t.free(b)
    with pytest.raises(KeyError):
        t.length(b)
    with pytest.raises(ValueError):
        t.fork(a, -1)
    for n, page in ((0, 16), (4, 8), (4, 24), (4, 8192)):
        with pytest.raises(ValueError, match="power of two"):
            PageTable(n, page)
    with pytest.raises(ValueError, match="32 bits"):
        PageTable(1 << 20, 2048)
    with pytest.raises(ValueError, match="precision"):
        PagedKVCache("cpu", 1, 2, 64, 4, precision="fp8")
    with pytest.raises(ValueError, match="layers"):
        PagedKVCache("cpu", 0, 2, 64, 4)


def test_cache_on_the_host():
    """The device arrays of a batch, here in host memory."""
    cache = PagedKVCache("cpu", 2, 2, 64, 8, 16, "bf16")
    a = cache.add()
    batch = cache.extend([a], [33])
    assert batch.fresh and batch.tokens == 33 and batch.end == 33 and batch.prefix_len == 0
    assert batch.starts.tolist() == [0, 33] and batch.tables.shape == (0, 0) and batch.lengths.numel() == 0
    batch = cache.extend([a])
    assert not batch.fresh and batch.prefix_len == 32 and batch.lengths.tolist() == [2] and batch.positions.tolist() == [33]
    assert cache.layer(1)[1].data_ptr() == cache.pool[3].data_ptr() and cache.length(a) == 34
    assert cache.stats()["resident_bytes"] == cache.pool.numel() * 2
    with pytest.raises(IndexError):
        cache.layer(2)
    with pytest.raises(ValueError, match="batch of 1 tokens"):
        BatchedAttention(AttentionConfig(128, 4, 2, 64)).forward(0, torch.zeros((3, 128)), {}, batch, cache)


def test_rope_tables_are_rope_cos_sin(monkeypatch):
    class Stream:
        def synchronize(self):
            pass

    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream())
    cfg = AttentionConfig(128, 4, 2, 64, rope_factor=32.0)
    att = BatchedAttention(cfg)
    cpu = torch.device("cpu")
    cos, sin = att.rope_tables(10, cpu)
    assert cos.shape == (1024, 32) and att.rope_tables(1024, cpu)[0] is cos
    more = att.rope_tables(1025, cpu)
    assert more[0].shape == (2048, 32) and torch.equal(more[1][:1024], sin)
    for p in (0, 1, 777, 2047):
        want = rope_cos_sin(cfg, p, cpu, torch.bfloat16)
        assert torch.equal(more[0][p], want[0]) and torch.equal(more[1][p], want[1])
