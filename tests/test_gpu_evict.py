"""Eviction of the keys of least weight from pages, against the definition: places, weights, keys and values exact."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from klcquant_amd import ops
from oracle import chunk

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def int32(values, gpu):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device=gpu)


class Caches:
    def __init__(self, gpu, lengths, layers=2, kv=2, dim=64, page=16, dtype="fp16", seed=0, capacity=None, weights=None):
        r = np.random.RandomState(seed)
        self.page, self.lengths = page, lengths
        held = [-(-max(n, 0) // page) for n in lengths]
        n_pages = sum(held) + 2
        order = r.permutation(n_pages)
        self.tables = np.full((len(lengths), max(held) + 1), -1)
        for b, h in enumerate(held):
            self.tables[b, :h] = order[sum(held[:b]):sum(held[:b]) + h]
        self.pools = torch.randint(-2 ** 15, 2 ** 15, (2 * layers, n_pages, page, kv, dim), dtype=torch.int16, device=gpu).view(DTYPES[dtype])
        capacity = capacity or (max(held) + 1) * page
        self.rows = r.permutation(len(lengths) + 1)[:len(lengths)]
        if weights is None:
            weights = r.standard_normal((layers, len(lengths) + 1, kv, capacity)).astype(np.float32)
            weights[:, :, 0] = np.floor(weights[:, :, 0] * 2)  # many alike, negative zeros among them
            weights[r.random_sample(weights.shape) < 0.2] = 0.0
        self.weights = torch.from_numpy(np.array(weights, dtype=np.float32)).to(gpu)
        self.gpu = gpu

    def run(self, keep, recent=0, first=0):
        self.before = self.pools.view(torch.int16).clone(), self.weights.cpu().numpy().copy()
        return ops.evict_keys(self.pools, self.weights, int32(self.tables, self.gpu), int32(self.lengths, self.gpu),
                              int32(self.rows, self.gpu), keep, recent=recent, first=first)

    def check(self, keep, recent=0, first=0):
        kept = self.run(keep, recent, first)
        pools, weights = self.before[0], self.before[1].copy()
        old = pools.cpu().numpy()
        want, got = old.copy(), self.pools.view(torch.int16).cpu().numpy()
        layers, kv = weights.shape[0], weights.shape[2]
        place = np.arange(keep)
        for layer in range(layers):
            for b, n in enumerate(self.lengths):
                for h in range(kv):
                    w = self.before[1][layer, self.rows[b], h]
                    at = chunk.kept_places(w, n, keep, recent, first)
                    assert (kept[layer, b, h].cpu().numpy() == at).all(), (layer, b, h)
                    if n <= keep:
                        continue
                    weights[layer, self.rows[b], h, :keep] = w[at]
                    t = self.tables[b]
                    for p in (2 * layer, 2 * layer + 1):
                        want[p, t[place // self.page], place % self.page, h] = old[p, t[at // self.page], at % self.page, h]
        assert (self.weights.cpu().numpy().view(np.int32) == weights.view(np.int32)).all()
        assert (got == want).all()
        return kept


@pytest.mark.parametrize("lengths,keep,recent,first", [
    ([1], 1, 0, 0), ([2], 1, 0, 0), ([2], 1, 1, 0), ([2], 1, 0, 1), ([40, 17, 3], 16, 4, 2), ([200, 100, 150], 100, 30, 4),
    ([2064, 2000, 1990], 2000, 128, 4), ([3000], 1, 1, 0), ([3000], 2999, 0, 0), ([3000, 2500], 2400, 2400, 0),
    ([3000, 2500], 1000, 500, 500), ([3000], 1000, 0, 1000), ([1025, 1024, 1023], 1000, 24, 0), ([5000, 0, -1], 70, 64, 3),
    ([2100], 2000, 1999, 1), ([4097], 2048, 1030, 0)])
def test_places(gpu, lengths, keep, recent, first):
    Caches(gpu, lengths).check(keep, recent, first)


@pytest.mark.parametrize("layers,kv,dim,page,dtype", [(1, 8, 64, 64, "bf16"), (3, 1, 128, 16, "fp16"), (2, 5, 48, 32, "fp16"),
                                                      (1, 4, 96, 128, "bf16"), (2, 3, 8, 16, "fp16"), (1, 2, 120, 16, "bf16")])
def test_shapes(gpu, layers, kv, dim, page, dtype):
    Caches(gpu, [700, 300, 33], layers, kv, dim, page, dtype, seed=dim).check(250, 50, 7)


def test_weights_alike(gpu):
    """Equal weights stay from the lowest place on; the zeros of both signs are equal."""
    for value in (0.0, -0.0, 3.5, -1.0, math.inf, -math.inf, math.nan, 1e-45):
        c = Caches(gpu, [900], weights=np.full((2, 2, 2, 1000), value))
        kept = c.check(400, 100, 4)
        assert (kept[..., :300].cpu() == torch.arange(300)).all()
    w = np.zeros((1, 2, 2, 600), np.float32)
    w[..., ::2] = -0.0
    kept = Caches(gpu, [600], layers=1, weights=w).check(100, 0, 0)
    assert (kept.cpu() == torch.arange(100)).all()


def test_special_weights(gpu):
    r = np.random.RandomState(4)
    w = r.standard_normal((2, 3, 2, 1500)).astype(np.float32)
    for value, share in ((math.nan, 0.05), (math.inf, 0.05), (-math.inf, 0.2), (1e-42, 0.1), (-1e-42, 0.1), (3.4e38, 0.02)):
        w[r.random_sample(w.shape) < share] = value
    w.view(np.uint32)[0, 0, 0, 100] = 0xFFC00001  # a NaN with its sign
    Caches(gpu, [1400, 900], weights=w).check(600, 64, 2)


def test_cut_again(gpu):
    """What was cut is cut further, and grows between."""
    c = Caches(gpu, [900, 800])
    c.check(500, 40, 4)
    c.lengths = [560, 520]
    c.check(500, 40, 4)
    c.lengths = [501, 500]
    c.check(500, 40, 4)
    c.check(100, 100, 0)


def test_what_is_left_alone(gpu):
    """Lengths past the tables or the weights, rows outside them, pages outside the pool, other layers' rows."""
    c = Caches(gpu, [300, 300, 300], capacity=304)
    c.lengths = [305, 300, 10 ** 9]
    kept = c.run(100, 10, 2)
    assert (kept[:, 0] == -1).all() and (kept[:, 2] == -1).all() and (kept[:, 1] >= 0).all()
    same = np.ones(c.before[1].shape, bool)
    same[:, c.rows[1], :, :100] = False
    assert (c.weights.cpu().numpy().view(np.int32)[same] == c.before[1].view(np.int32)[same]).all()
    touched = (c.pools.view(torch.int16) != c.before[0]).any(dim=4).any(dim=3).any(dim=0)
    assert set(touched.any(dim=1).nonzero().flatten().tolist()) <= set(c.tables[1][:7].tolist())
    c = Caches(gpu, [300, 300])
    c.rows = np.array([3, -1])
    kept = c.run(100, 10, 2)
    assert (kept == -1).all() and torch.equal(c.pools.view(torch.int16), c.before[0])
    c = Caches(gpu, [300, 300])
    c.tables[0, 15], c.tables[0, 2], c.tables[0, 1] = -1, c.pools.shape[1], 2 ** 31 - 1
    c.run(100, 10, 2)
    touched = (c.pools.view(torch.int16) != c.before[0]).any(dim=4).any(dim=3).any(dim=0).any(dim=1)
    assert set(touched.nonzero().flatten().tolist()) <= set(c.tables[0, [0, 3, 4, 5, 6]].tolist()) | set(c.tables[1, :7].tolist())


def test_no_sequences_and_no_pages(gpu):
    c = Caches(gpu, [40])
    empty = torch.zeros((0, 3), dtype=torch.int32, device=gpu)
    none = torch.zeros(0, dtype=torch.int32, device=gpu)
    assert ops.evict_keys(c.pools, c.weights, empty, none, none, 4).shape == (2, 0, 2, 4)
    one = torch.zeros(1, dtype=torch.int32, device=gpu)
    assert (ops.evict_keys(c.pools, c.weights, torch.zeros((1, 0), dtype=torch.int32, device=gpu), one, one, 4) == -1).all()


def test_captured_and_replayed(gpu):
    c, e = Caches(gpu, [900, 700], seed=2), Caches(gpu, [900, 700], seed=2)
    e.pools.copy_(c.pools)
    tables, lengths, rows = int32(c.tables, gpu), int32(c.lengths, gpu), int32(c.rows, gpu)
    c.run(899, 0, 0)
    e.run(899, 0, 0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = ops.evict_keys(c.pools, c.weights, tables, lengths, rows, 300, recent=32, first=1)
    for n in (800, 650, 400, 301):
        for x in (c, e):
            x.weights.copy_(torch.randn(x.weights.shape, generator=torch.Generator().manual_seed(n)).to(gpu))
        lengths.fill_(n)
        graph.replay()
        torch.cuda.synchronize()
        e.lengths = [n, n]
        want = e.run(300, 32, 1)
        assert torch.equal(kept, want) and torch.equal(c.weights, e.weights)
        assert torch.equal(c.pools.view(torch.int16), e.pools.view(torch.int16))


def test_long_lists(gpu):
    """More keys than a pass of the workgroup over many times, in one KV head."""
    c = Caches(gpu, [70000], layers=1, kv=1, dim=16, page=256)
    c.check(30000, 3000, 100)
    c.lengths = [30000]
    c.check(29990, 20000, 0)


def test_past_32_bits(gpu):
    pages, page, kv, dim = 2300, 1024, 8, 128
    pools = torch.zeros((2, pages, page, kv, dim), dtype=torch.bfloat16, device=gpu)
    small = torch.randn((2, 3, page, kv, dim), device=gpu).bfloat16()
    far = [2299, 1, 2298]
    pools[:, far] = small
    w = torch.rand((1, 1, kv, 3 * page), device=gpu)
    w2 = w.clone()
    n, row = int32([3000], gpu), int32([0], gpu)
    a = ops.evict_keys(pools, w, int32([far], gpu), n, row, 1100, recent=100)
    b = ops.evict_keys(small, w2, int32([[0, 1, 2]], gpu), n, row, 1100, recent=100)
    assert torch.equal(a, b) and torch.equal(w, w2) and torch.equal(pools[:, far], small)
