"""Key weights of batches whose sequences differ much, and of lengths that are far from those the plan was made for: right
against their definition in float64, with scratch memory that goes by what each sequence's own new tokens see."""

from __future__ import annotations

import pytest
import torch

from klcquant_amd import ops
from test_gpu_chunk_attention import Case, int32

pytestmark = pytest.mark.gpu


def scratch_bytes(call):
    """What a call allocates beyond what is held before and after it."""
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    call()
    torch.cuda.synchronize()
    return torch.cuda.max_memory_allocated() - before


@pytest.mark.parametrize("counts,keys,window,first", [
    ([100] * 24 + [1], [600] * 24 + [60000], None, 0), ([500] * 12 + [1], [900] * 12 + [60000], 128, 4)])
def test_suffixes_beside_one_long_sequence(gpu, counts, keys, window, first):
    """Not a row of scratch over the longest sequence's keys for every part of the others' rows (24 x 60,000 x 8 x 8
    bytes and more): blocks of 256 keys x 8 x 8 bytes, one for each that is seen and 512 more."""
    c = Case(gpu, "fp16", 64, 8, 64, 64, counts, keys, window, first)
    _, lse = c.run(want_lse=True)
    weights = torch.zeros((len(counts), 8, 60032), device=gpu)
    rows = torch.arange(len(counts), dtype=torch.int32, device=gpu)
    used = scratch_bytes(lambda: ops.add_key_weights(c.q, lse, c.k, c.table, c.lengths, c.plan, weights, rows))
    assert used <= 2048 * 8 * (sum(-(-n // 256) for n in keys) + 512 + 1)
    del weights
    c.check_weights(lse)


@pytest.mark.parametrize("window,first", [(None, 0), (100, 0), (100, 4), (300, 270)])
@pytest.mark.parametrize("heads,kv,dim,dtype", [(16, 4, 64, "fp16"), (8, 1, 128, "bf16"), (6, 2, 96, "fp16")])
def test_far_from_the_planned_lengths(gpu, heads, kv, dim, dtype, window, first):
    """Sequences that have grown by many blocks of keys, in parts of rows and whole, and shorter ones."""
    counts, keys = [1, 600, 6, 300], [3000, 2600, 800, 300]
    c = Case(gpu, dtype, heads, kv, dim, 64, counts, keys, window, first)
    _, lse = c.check()
    for planned in (counts, [n + 2000 for n in keys], [300, 5000, 6, 301], keys):
        c.plan = ops.attention_plan(counts, planned, heads, kv, dim, window, first)
        c.check_weights(lse)


@pytest.mark.parametrize("window,first", [(None, 0), (40, 0), (40, 4), (40, 300)])
def test_bad_pages_and_lengths_touch_what_is_seen(gpu, window, first):
    """A page outside the pool makes the weights NaN of its keys that some new token sees, whichever others share their
    block of 256, and so does a length past the table; the others keep theirs."""
    keys, new, page = [900, 700], [1, 30], 16
    c = Case(gpu, "fp16", 8, 2, 64, page, new, keys, window, first)
    _, lse = c.run(want_lse=True)
    rows = int32([0, 1], gpu)

    def seen(n, count):
        at = torch.arange(n, device=gpu)
        return at >= 0 if window is None else (at > n - count - window) | (at < first)

    bad = [0, 3, 17, 30, 41, 42, 43, 54, 55, 56]
    for number in (-1, c.k.shape[0], 2 ** 31 - 1, -2 ** 31):
        table = c.table.clone()
        for p in bad:
            table[:, p] = torch.where(table[:, p] >= 0, number, table[:, p])
        weights = torch.full((2, 2, 1024), 7.0, device=gpu)
        ops.add_key_weights(c.q, lse, c.k, table, c.lengths, c.plan, weights, rows)
        for b, n in enumerate(keys):
            at = torch.arange(n, device=gpu)
            hit = seen(n, new[b]) & torch.isin(at // page, torch.tensor(bad, device=gpu))
            assert hit.any() and torch.equal(weights[b, :, :n].isnan(), hit.expand(2, n))
            assert (weights[b, :, :n][:, ~seen(n, new[b])] == 7).all() and (weights[b, :, n:] == 7).all()
    room = c.width * page
    c.lengths[0] = room + 1
    weights = torch.full((2, 2, 1024), 7.0, device=gpu)
    ops.add_key_weights(c.q, lse, c.k, c.table, c.lengths, c.plan, weights, rows)
    assert torch.equal(weights[0, :, :room].isnan(), seen(room, 1).expand(2, room)) and torch.isfinite(weights[1]).all()
    assert (weights[0, :, :room][:, ~seen(room, 1)] == 7).all() and (weights[0, :, room:] == 7).all()


def test_two_streams_and_one_plan(gpu):
    c = Case(gpu, "bf16", 8, 2, 64, 64, [2, 900], [6000, 2000])
    assert c.plan.list_joins > 0
    _, lse = c.run(want_lse=True)
    rows = int32([1, 0], gpu)
    weights = [torch.zeros((2, 2, 6016), device=gpu) for _ in range(7)]
    streams = [torch.cuda.Stream(gpu) for _ in range(2)]
    torch.cuda.synchronize()
    for i, w in enumerate(weights):
        with torch.cuda.stream(streams[i % 2]):
            ops.add_key_weights(c.q, lse, c.k, c.table, c.lengths, c.plan, w, rows)
    torch.cuda.synchronize()
    assert weights[0].any() and all(torch.equal(w, weights[0]) for w in weights)


def test_a_plan_without_key_weights(gpu):
    c = Case(gpu, "bf16", 8, 2, 64, 64, [2], [100])
    _, lse = c.run(want_lse=True)
    plan = ops.attention_plan([2], [100], 8, 2, 64, key_weights=False)
    assert plan.data.numel() < c.plan.data.numel()
    assert torch.equal(ops.chunk_attention(c.q, c.k, c.v, c.table, c.lengths, plan), c.run())
    with pytest.raises(ValueError, match="key_weights"):
        ops.add_key_weights(c.q, lse, c.k, c.table, c.lengths, plan, torch.zeros((1, 2, 128), device=gpu), int32([0], gpu))


@pytest.mark.parametrize("window,first", [(None, 0), (100, 4)])
def test_captured_and_replayed_over_many_blocks(gpu, window, first):
    """A graph whose sequences grow past the blocks of keys that its list was made for: as a list made for each length."""
    counts, keys = [1, 300], [2400, 2600]
    c = Case(gpu, "fp16", 16, 4, 64, 64, counts, keys, window, first)
    rows = int32([1, 0], gpu)
    lengths = [[200 + 700 * i, 310 + 700 * i] for i in range(4)]
    weights = torch.zeros((2, 4, 2688), device=gpu)
    c.lengths.copy_(int32(lengths[0], gpu))
    plan = ops.attention_plan(counts, lengths[0], 16, 4, 64, window, first)
    _, lse = ops.chunk_attention(c.q, c.k, c.v, c.table, c.lengths, plan, want_lse=True)
    ops.add_key_weights(c.q, lse, c.k, c.table, c.lengths, plan, weights, rows)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, lse = ops.chunk_attention(c.q, c.k, c.v, c.table, c.lengths, plan, want_lse=True)
        ops.add_key_weights(c.q, lse, c.k, c.table, c.lengths, plan, weights, rows)
    for now in (lengths[1], lengths[3], lengths[0], lengths[2]):
        c.lengths.copy_(int32(now, gpu))
        weights.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = weights.clone()
        again = ops.attention_plan(counts, now, 16, 4, 64, window, first)
        want, norm = torch.zeros_like(weights), ops.chunk_attention(c.q, c.k, c.v, c.table, c.lengths, again, want_lse=True)[1]
        ops.add_key_weights(c.q, norm, c.k, c.table, c.lengths, again, want, rows)
        # the logs by other parts of the keys, 2^-20 of each weight, and sums of the same float32 sums in float64
        assert torch.isfinite(got).all() and got.any() and torch.allclose(got, want, rtol=1e-5, atol=1e-30)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("factor", [2.0 ** 60, 2.0 ** -60])
def test_queries_of_all_sizes(gpu, dtype, factor):
    """A power of two more in the queries and less in the scale changes no bit of the weights."""
    c = Case(gpu, dtype, 8, 2, 64, 16, [3, 40], [50, 390])
    _, lse = c.run(want_lse=True)
    rows, weights = int32([0, 1], gpu), torch.zeros((2, 2, 2, 400), device=gpu)
    ops.add_key_weights(c.q, lse, c.k, c.table, c.lengths, c.plan, weights[0], rows)
    ops.add_key_weights(c.q * factor, lse, c.k, c.table, c.lengths, c.plan, weights[1], rows, scale=c.scale / factor)
    assert weights[0].any() and torch.equal(weights[0], weights[1])
