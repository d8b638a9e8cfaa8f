"""Attention of chunks of new tokens over pages, and the weights that they give the keys, against their definition in
float64.  Tolerances: oracle.prompt.tolerance for the results; for the logs of the normalisers and for the weights the
float32 work on the scores, sums and logs, counted below."""

from __future__ import annotations

import math

import pytest
import torch

from klcquant_amd import ops
from oracle import chunk, prompt

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def int32(values, gpu):
    return torch.tensor(values, dtype=torch.int32, device=gpu)


class Case:
    """Sequences of counts[s] new tokens among keys[s] in scattered pages; every page that none holds is NaN."""

    def __init__(self, gpu, dtype, heads, kv, dim, page, counts, keys, window=None, first=0, sinks=False, seed=0, std=1.0,
                 fused=False, spare=2):
        g = torch.Generator(device=gpu).manual_seed(seed + dim + sum(keys))
        self.gpu, self.counts, self.keys, self.window, self.first = gpu, counts, keys, window, first
        held = [-(-n // page) for n in keys]
        order = torch.randperm(sum(held) + spare, generator=torch.Generator().manual_seed(seed)).tolist()
        self.tables = [order[sum(held[:b]):sum(held[:b + 1])] for b in range(len(keys))]
        self.width = max(held) + 1
        self.table = int32([t + [-1] * (self.width - len(t)) for t in self.tables], gpu)
        self.lengths = int32(keys, gpu)
        tokens = sum(counts)
        q = torch.randn((tokens, heads + (8 if fused else 0), dim), device=gpu, generator=g).mul_(std).bfloat16()
        self.q = q[:, :heads]
        self.k, self.v = (torch.full((sum(held) + spare, page, kv, dim), math.nan, dtype=DTYPES[dtype], device=gpu) for _ in range(2))
        for b, n in enumerate(keys):
            at = torch.tensor([self.tables[b][i // page] * page + i % page for i in range(n)], dtype=torch.long, device=gpu)
            for x in (self.k, self.v):
                x.view(-1, kv, dim)[at] = torch.randn((n, kv, dim), device=gpu, generator=g).to(DTYPES[dtype])
        self.sinks = torch.randn(heads, device=gpu, generator=g).bfloat16() if sinks else None
        self.plan = ops.attention_plan(counts, keys, heads, kv, dim, window, first)
        self.scale = dim ** -0.5
        self.starts = [sum(counts[:b]) for b in range(len(counts) + 1)]

    def run(self, **more):
        return ops.chunk_attention(self.q, self.k, self.v, self.table, self.lengths, self.plan, sinks=self.sinks, **more)

    def want(self, b):
        """(rows of sequence b, the oracle's answer)"""
        n, count = int(self.lengths[b]), self.counts[b]
        rows = torch.arange(n - count, n, device=self.gpu)
        k, v = (chunk.gather(x, self.tables[b], n) for x in (self.k, self.v))
        at = slice(self.starts[b], self.starts[b + 1])
        return at, chunk.attend(self.q[at], k, v, rows, self.sinks, self.window, self.first, self.scale)

    def score_error(self, at, reach):
        """What float32 sums of products add to a score, and in a float16 cache small elements of the query."""
        q = self.q[at].double().abs().amax(dim=2)
        most = torch.nan_to_num(self.k.float(), nan=0.0, posinf=0.0, neginf=0.0).abs().sum(dim=3).amax()
        small = 2.0 ** -25 * q * float(most) * self.scale if self.k.dtype == torch.float16 else 0.0
        return 2 * (self.q.shape[2] + 4) * 2.0 ** -24 * reach + small

    def check(self, only=None):
        out, lse = self.run(want_lse=True)
        assert torch.equal(self.run().nan_to_num(nan=77.0), out.nan_to_num(nan=77.0))
        for b in range(len(self.counts)) if only is None else only:
            at, (want, norm, _, size, reach) = self.want(b)
            n = int(self.lengths[b])
            v_most = float(torch.nan_to_num(self.v.float(), nan=0.0, posinf=0.0, neginf=0.0).abs().max())
            assert torch.equal(out[at].isnan(), want.isnan()), b
            tol = prompt.tolerance(want, size, reach, n, self.q.shape[2], self.k.dtype, torch.bfloat16, v_most)
            off = ((out[at].double() - want).abs() / tol).nan_to_num(nan=0.0)
            inf = torch.isinf(want)
            assert torch.equal(out[at].double()[inf], want[inf])
            assert float(off[~inf].max() if (~inf).any() else 0.0) <= 1.0, (b, float(off[~inf].max()))
            fine = torch.isfinite(norm)
            assert torch.equal(lse[at].double()[~fine].nan_to_num(nan=77.0), norm[~fine].nan_to_num(nan=77.0)), b
            # scores, the sum's roundings, and those of the logarithm, its base and their products
            tol = self.score_error(at, reach) + (n + 64) * 2.0 ** -24 + 6 * 2.0 ** -24 * (norm.abs() + 1)
            assert float(((lse[at].double() - norm).abs() / tol)[fine].max() if fine.any() else 0.0) <= 1.0, b
        return out, lse

    def check_weights(self, lse, capacity=None):
        kv = self.k.shape[2]
        capacity = capacity or self.width * self.k.shape[1]
        g = torch.Generator(device=self.gpu).manual_seed(5)
        rows = torch.randperm(len(self.counts) + 2, device=self.gpu, generator=g)[:len(self.counts)].int()
        weights = torch.rand((len(self.counts) + 2, kv, capacity), device=self.gpu, generator=g)
        before = weights.double()
        ops.add_key_weights(self.q, lse, self.k, self.table, self.lengths, self.plan, weights, rows)
        left = torch.ones(weights.shape, dtype=torch.bool, device=self.gpu)
        for b, count in enumerate(self.counts):
            at, (_, norm, w, _, reach) = self.want(b)
            n = int(self.lengths[b])
            group = self.q.shape[1] // kv
            want = w.view(count, kv, group, n).sum(dim=(0, 2))
            row = int(rows[b])
            start = before[row, :, :n].clone()
            start[:, max(0, n - count):] = 0.0
            # of each weight: its score's error and lse's, twice for the exponential's own; 64 sums of a tile; the result
            share = (self.score_error(at, reach) * 2 + 16 * 2.0 ** -24 * (norm.abs() + 1) + (n + 128) * 2.0 ** -24)
            share = share.nan_to_num(nan=0.0, posinf=0.0, neginf=0.0)[:, :, None]
            tol = (w.nan_to_num(nan=0.0) * share).view(count, kv, group, n).sum(dim=(0, 2)) + 2.0 ** -23 * (start + want.abs()) + 1e-37
            got = weights[row, :, :n].double()
            assert torch.equal(got.isnan(), (start + want).isnan()), b
            off = ((got - start - want).abs() / tol).nan_to_num(nan=0.0)
            assert float(off.max()) <= 1.0, (b, float(off.max()))
            left[row, :, :n] = False
        assert torch.equal(weights.double()[left], before[left])  # other rows, and places behind the keys
        return weights


SHAPES = [(64, 8, 64, 64), (32, 8, 128, 16), (28, 4, 80, 32), (8, 1, 128, 64), (3, 3, 64, 16), (20, 5, 48, 16), (24, 4, 96, 64),
          (40, 1, 64, 16), (2, 1, 8, 16), (16, 4, 40, 128)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("heads,kv,dim,page", SHAPES)
def test_one_token_and_many(gpu, dtype, heads, kv, dim, page):
    """One key; one token behind many; a whole prompt; suffixes that start and end inside tiles and pages."""
    counts, keys = [1, 1, 50, 7, 33, 1], [1, 130, 50, 75, 301, 64]
    c = Case(gpu, dtype, heads, kv, dim, page, counts, keys, sinks=dim % 3 == 0)
    _, lse = c.check()
    c.check_weights(lse)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("heads,kv,dim,page", [(64, 8, 64, 64), (8, 2, 128, 16), (6, 2, 24, 16)])
@pytest.mark.parametrize("window,first", [(1, 0), (1, 1), (16, 3), (100, 4), (100, 90), (37, 64), (5000, 2)])
def test_windows_and_first_tokens(gpu, dtype, heads, kv, dim, page, window, first):
    counts, keys = [1, 1, 40, 4, 1, 150, 90], [1, 400, 40, 303, 50, 350, 90]
    c = Case(gpu, dtype, heads, kv, dim, page, counts, keys, window, first, sinks=window == 16)
    _, lse = c.check()
    c.check_weights(lse)


@pytest.mark.parametrize("heads,kv,dim,dtype", [(8, 2, 64, "fp16"), (8, 2, 128, "bf16"), (4, 4, 64, "bf16"), (7, 1, 96, "fp16")])
@pytest.mark.parametrize("counts,keys", [([1], [9000]), ([3], [6001]), ([257], [5000]), ([1, 600], [3500, 4100])])
def test_keys_in_parts(gpu, heads, kv, dim, dtype, counts, keys):
    """Few rows over many keys: parts that are joined, and waves that share a token's keys."""
    c = Case(gpu, dtype, heads, kv, dim, 64, counts, keys, sinks=True)
    assert c.plan.joins > 0
    _, lse = c.check()
    c.check_weights(lse)


@pytest.mark.parametrize("window,first", [(None, 0), (100, 0), (100, 4), (300, 270)])
def test_weights_of_rows_in_parts(gpu, window, first):
    """A long chunk beside steps: parts that some blocks of keys have no rows for."""
    c = Case(gpu, "fp16", 16, 4, 64, 16, [1, 700, 5, 90], [800, 1500, 5, 1000], window, first)
    assert c.plan.weight_joins > 0 and c.plan.weight_parts > 2 * c.plan.weight_joins
    _, lse = c.check()
    c.check_weights(lse)


def test_one_long_sequence_among_many(gpu):
    c = Case(gpu, "fp16", 8, 8, 64, 64, [1] * 130, [100 + i for i in range(129)] + [20000])
    assert 0 < c.plan.joins < 130
    _, lse = c.check(only=(0, 64, 128, 129))


def test_a_fused_projection_and_out(gpu):
    c = Case(gpu, "fp16", 16, 4, 64, 16, [5, 1, 90], [60, 200, 91], fused=True)
    assert not c.q.is_contiguous()
    out, lse = c.check()
    c.check_weights(lse)
    held = torch.empty_like(out)
    assert c.run(out=held) is held and torch.equal(held, out)


def test_queries_of_all_sizes(gpu):
    """A float16 cache takes bfloat16 queries past float16's range."""
    c = Case(gpu, "fp16", 8, 2, 64, 16, [3, 40], [50, 90])
    for factor in (2.0 ** 60, 2.0 ** -60):
        c.q = c.q * factor
        c.scale = 1 / (factor * 8)
        out, lse = ops.chunk_attention(c.q, c.k, c.v, c.table, c.lengths, c.plan, scale=c.scale, want_lse=True)
        for b in range(2):
            at, (want, norm, _, size, reach) = c.want(b)
            tol = prompt.tolerance(want, size, reach, 90, 64, torch.float16, torch.bfloat16, float(torch.nan_to_num(c.v.float()).abs().max()))
            assert float(((out[at].double() - want).abs() / tol).max()) <= 1.0
            assert float((lse[at].double() - norm).abs().max()) <= 1e-4
        c.q = c.q / factor


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("heads,kv,dim", [(64, 8, 64), (8, 2, 128), (4, 1, 40)])
@pytest.mark.parametrize("window,first", [(None, 0), (20, 3)])
def test_nan_and_infinity_reach_only_those_that_see_them(gpu, dtype, heads, kv, dim, window, first):
    counts, keys = [60, 3, 1, 400], [90, 40, 70, 3000]
    c = Case(gpu, dtype, heads, kv, dim, 16, counts, keys, window, first)
    clean = c.run()
    k, v = c.k.view(-1, kv, dim), c.v.view(-1, kv, dim)
    slot = lambda b, i: c.tables[b][i // 16] * 16 + i % 16  # noqa: E731
    # of new tokens in the middle of the chunk, and of the first key behind a window
    v[slot(0, 60), 0, 1], v[slot(0, 75), kv - 1, dim - 1] = math.inf, math.nan
    v[slot(1, 39), 0, 0] = -math.inf
    k[slot(0, 80), 0] = math.nan
    v[slot(3, 2800), 0, 3] = math.inf
    k[slot(3, 2990), 0, 0] = math.nan
    v[slot(2, 10), 0, 0] = math.nan
    out, lse = c.check()
    # sequence 0's tokens before key 60 see nothing of it
    assert torch.equal(out[:30], clean[:30])
    weights = c.check_weights(lse)
    assert weights.isnan().any()


def test_scores_of_minus_infinity(gpu):
    """Scores that are all -inf: NaN without a sink, nothing with one.  A row without a key is zero."""
    c = Case(gpu, "bf16", 8, 2, 64, 16, [20, 1], [20, 500])
    c.q[..., 0] = c.q[..., 0].abs() + 1
    page = c.k.shape[1]
    for b, n in ((0, 5), (1, 500)):
        for i in range(n):
            c.k[c.tables[b][i // page], i % page, :, 0] = -math.inf
    out, lse = c.check()
    assert out[:5].isnan().all() and torch.isfinite(out[5:20]).all() and out[20].isnan().all() and (lse[20] == -math.inf).all()
    c.sinks = torch.zeros(8, dtype=torch.bfloat16, device=gpu)
    out, lse = c.run(want_lse=True)
    assert not out[:5].any() and not out[20].any() and torch.isfinite(out).all() and not lse[20].any()


def test_lengths_that_are_not_the_plans(gpu):
    """Longer and shorter sequences than planned, as a replayed step's; tokens without a place in them are zero."""
    c = Case(gpu, "fp16", 16, 4, 64, 16, [1, 6, 70], [100, 80, 300])
    c.plan = ops.attention_plan(c.counts, [1, 6, 70], 16, 4, 64)
    _, lse = c.check()
    c.check_weights(lse)
    c.lengths = int32([37, 3, 69], gpu)
    out, lse = c.check()
    assert not out[1:4].any() and not out[7].any() and (lse[1:4] == -math.inf).all()
    c.check_weights(lse)
    for none in (0, -1, -2 ** 31):
        c.lengths = int32([none, 80, none], gpu)
        out, lse = c.run(want_lse=True)
        assert not out[0].any() and not out[7:].any() and out[1:7].any() and (lse[0] == -math.inf).all()
        weights = torch.ones((3, 4, 512), device=gpu)
        ops.add_key_weights(c.q, lse, c.k, c.table, c.lengths, c.plan, weights, int32([0, 1, 2], gpu))
        assert (weights[0] == 1).all() and (weights[2] == 1).all() and torch.isfinite(weights).all()


def test_bad_pages_and_lengths(gpu):
    """A page number outside the pool makes the rows that see it NaN; pages that none sees may be anything."""
    for window, first in ((None, 0), (40, 4)):
        c = Case(gpu, "fp16", 8, 2, 64, 16, [1, 30, 1], [300, 200, 250], window, first)
        clean, lse = c.check()
        for bad in (-1, c.k.shape[0], 2 ** 31 - 1, -2 ** 31):
            table = c.table.clone()
            table[0, 3] = bad
            table[1, 12] = bad
            out = ops.chunk_attention(c.q, c.k, c.v, table, c.lengths, c.plan)
            hidden = window is not None  # key 48 of 300
            assert out[0].isnan().all() != hidden and out[30].isnan().all() and torch.equal(out[31], clean[31])
            assert not hidden or torch.equal(out[0], clean[0])
            weights = torch.zeros((3, 2, 400), device=gpu)
            ops.add_key_weights(c.q, lse, c.k, table, c.lengths, c.plan, weights, int32([0, 1, 2], gpu))
            assert weights[1, :, 192:200].isnan().all() and torch.isfinite(weights[1, :, :192]).all()
            assert torch.isfinite(weights[2]).all()
        c.lengths[0] = c.width * 16 + 1
        out = c.run()
        assert out[0].isnan().all() and torch.equal(out[1:], clean[1:])


def test_weights_left_out(gpu):
    """Keys past the capacity, and rows outside the weights."""
    c = Case(gpu, "bf16", 8, 2, 64, 16, [1, 5], [100, 60])
    _, lse = c.check()
    full = torch.zeros((2, 2, 128), device=gpu)
    ops.add_key_weights(c.q, lse, c.k, c.table, c.lengths, c.plan, full, int32([0, 1], gpu))
    part = torch.zeros((2, 2, 70), device=gpu)
    ops.add_key_weights(c.q, lse, c.k, c.table, c.lengths, c.plan, part, int32([0, -1], gpu))
    assert torch.equal(part[0], full[0, :, :70]) and not part[1].any()
    ops.add_key_weights(c.q, lse, c.k, c.table, c.lengths, c.plan, part, int32([2, 2 ** 31 - 1], gpu))
    assert torch.equal(part[0], full[0, :, :70]) and not part[1].any()


def test_the_same_every_time(gpu):
    c = Case(gpu, "fp16", 8, 1, 64, 64, [1, 300], [5000, 4000])
    out, lse = c.run(want_lse=True)
    rows = int32([1, 0], gpu)
    first = torch.zeros((2, 1, 5056), device=gpu)
    ops.add_key_weights(c.q, lse, c.k, c.table, c.lengths, c.plan, first, rows)
    for _ in range(5):
        again, norm = c.run(want_lse=True)
        weights = torch.zeros_like(first)
        ops.add_key_weights(c.q, lse, c.k, c.table, c.lengths, c.plan, weights, rows)
        assert torch.equal(again, out) and torch.equal(norm, lse) and torch.equal(weights, first)


def test_captured_and_replayed(gpu):
    """A step of parts and one of rows, captured, and replayed as the sequences grow and the queries change."""
    c = Case(gpu, "fp16", 8, 2, 64, 64, [1, 90], [4000, 700])
    rows = int32([0, 1], gpu)
    weights = torch.zeros((2, 2, 4160), device=gpu)
    keys = [4000 + 64, 700 + 64]
    extra = Case(gpu, "fp16", 8, 2, 64, 64, [1, 90], keys, seed=3)
    c.k, c.v, c.table, c.tables = extra.k, extra.v, extra.table, extra.tables
    weights.zero_()
    c.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = c.run(want_lse=True)
        ops.add_key_weights(c.q, lse, c.k, c.table, c.lengths, c.plan, weights, rows)
    for i in range(4):
        c.lengths += 13
        c.q.copy_(torch.randn_like(c.q))
        weights.zero_()
        out.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        got = weights.clone()
        want, norm = c.run(want_lse=True)
        weights.zero_()
        ops.add_key_weights(c.q, norm, c.k, c.table, c.lengths, c.plan, weights, rows)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, norm) and torch.equal(got, weights) and torch.isfinite(out).all()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ops.attention_plan([1], [5], 8, 2, 64)


def test_two_streams_and_one_plan(gpu):
    """Calls at once over one plan: workspaces of their own."""
    c = Case(gpu, "bf16", 8, 2, 128, 64, [2, 300], [6000, 2000])
    want = c.run()
    streams = [torch.cuda.Stream(gpu) for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(c.run())
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_past_32_bits(gpu):
    """Pages whose bytes and elements lie past 2^31 and 2^32."""
    pages, page, kv, dim = 2300, 1024, 8, 128
    k, v = (torch.zeros((pages, page, kv, dim), dtype=torch.bfloat16, device=gpu) for _ in range(2))
    c = Case(gpu, "bf16", 16, kv, dim, page, [1, 40], [1500, 1100], spare=0)
    far = [2299, 2290, 5, 2200]
    for b, t in enumerate(c.tables):
        for i, p in enumerate(t):
            k[far[2 * b + i]], v[far[2 * b + i]] = c.k[p].nan_to_num(nan=0.0), c.v[p].nan_to_num(nan=0.0)
    table = int32([[2299, 2290, -1], [5, 2200, -1]], gpu)
    want, lse = c.check()
    out = ops.chunk_attention(c.q, k, v, table, c.lengths, c.plan)
    assert torch.equal(out, want)
    weights = [torch.zeros((2, kv, 2048), device=gpu) for _ in range(2)]
    ops.add_key_weights(c.q, lse, c.k, c.table, c.lengths, c.plan, weights[0], int32([0, 1], gpu))
    ops.add_key_weights(c.q, lse, k, table, c.lengths, c.plan, weights[1], int32([0, 1], gpu))
    assert torch.equal(*weights)


def test_many_sequences(gpu):
    """More items than the chip holds, and rows behind others' in one tile list."""
    counts = [1 + (i * 7) % 5 if i % 3 else 1 for i in range(300)]
    keys = [c + (i * 37) % 190 for i, c in enumerate(counts)]
    c = Case(gpu, "fp16", 4, 2, 64, 16, counts, keys)
    _, lse = c.check(only=(0, 1, 2, 150, 298, 299))
    weights = torch.zeros((300, 2, 256), device=gpu)
    ops.add_key_weights(c.q, lse, c.k, c.table, c.lengths, c.plan, weights, torch.arange(300, dtype=torch.int32, device=gpu))
    # every row's weights sum up to one: no sinks
    sums = weights.double().sum(dim=(1, 2)).cpu()
    assert torch.allclose(sums, torch.tensor(counts, dtype=torch.float64) * 4, rtol=1e-5, atol=0)
