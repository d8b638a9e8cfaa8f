"""The paged cache's operators against their definitions: rotation and append, page copies, batch attention
(tolerances: oracle.prompt.tolerance; appends and copies exact up to the one rounding they name)."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from klcquant_amd import ops
from oracle import prompt

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def int32(values, gpu):
    return torch.tensor(values, dtype=torch.int32, device=gpu)


# ---- rotation and append ----------------------------------------------------------------


def rope_inputs(gpu, tokens, heads, kv, dim, seed=0, n_pos=5000, fused=False):
    g = torch.Generator(device=gpu).manual_seed(seed)
    x = torch.randn((tokens, heads + 2 * kv, dim), device=gpu, generator=g).bfloat16()
    q, k, v = x.split((heads, kv, kv), dim=1)
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    angle = torch.rand((n_pos, dim // 2), device=gpu, generator=g) * 6.3
    return q, k, v, angle.cos().bfloat16(), angle.sin().bfloat16()


def rotated(x, cos, sin, positions):
    a, b = x.double().chunk(2, dim=-1)
    c, s = cos.double()[positions][:, None], sin.double()[positions][:, None]
    return torch.cat((a * c - b * s, b * c + a * s), dim=-1)


def assert_rounded(got, want, dtype):
    """One float32 rounding of a sum of exact products, then one to the type (the smallest normal for subnormals)."""
    eps = torch.finfo(dtype).eps / 2
    off = want.abs() * (eps * (1 + 2.0 ** -23) + 2.0 ** -24) + torch.finfo(dtype).tiny * eps
    assert ((got.double() - want).abs() <= off).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("tokens,heads,kv,dim,fused", [(1, 64, 8, 64, False), (77, 64, 8, 64, True), (33, 7, 1, 80, False),
                                                       (300, 3, 3, 8, True), (5, 8, 2, 128, False), (19, 4, 1, 24, True)])
def test_append_rotates_and_stores(gpu, dtype, tokens, heads, kv, dim, fused):
    q, k, v, cos, sin = rope_inputs(gpu, tokens, heads, kv, dim, seed=tokens, fused=fused)
    page, n_pages = 16, 3 + tokens // 8
    g = torch.Generator().manual_seed(tokens)
    positions = torch.randint(0, 5000, (tokens,), generator=g).to(gpu)
    slots = torch.randperm(n_pages * page, generator=g)[:tokens].to(gpu)
    drop = tokens // 3  # tokens that are stored nowhere
    where = slots.clone()
    where[:drop] = torch.tensor([-1, n_pages * page, -2 ** 31, 2 ** 31 - 1], device=gpu)[torch.arange(drop, device=gpu) % 4]
    pools = [torch.full((n_pages, page, kv, dim), 9.0, dtype=DTYPES[dtype], device=gpu) for _ in range(2)]
    rq, rk = ops.paged_append(q, k, v, cos, sin, positions.int(), where.int(), *pools)
    wq, wk = rotated(q, cos, sin, positions), rotated(k, cos, sin, positions)
    assert_rounded(rq, wq, torch.bfloat16)
    assert_rounded(rk, wk, torch.bfloat16)
    flat_k, flat_v = (p.view(-1, kv, dim) for p in pools)
    assert_rounded(flat_k[slots[drop:]], wk[drop:], DTYPES[dtype])
    assert torch.equal(flat_v[slots[drop:]], v[drop:].float().to(DTYPES[dtype]))
    rest = torch.ones(n_pages * page, dtype=torch.bool, device=gpu)
    rest[slots[drop:]] = False
    assert (flat_k[rest] == 9).all() and (flat_v[rest] == 9).all()
    again, none = ops.paged_append(q, k, v, cos, sin, positions.int(), where.int(), *pools, want_keys=False)
    assert torch.equal(again, rq) and none is None


def test_append_position_outside_the_tables(gpu):
    q, k, v, cos, sin = rope_inputs(gpu, 4, 2, 1, 64, n_pos=10)
    pools = [torch.zeros((2, 16, 1, 64), dtype=torch.float16, device=gpu) for _ in range(2)]
    rq, rk = ops.paged_append(q, k, v, cos, sin, int32([9, 10, -1, 2 ** 31 - 1], gpu), int32([0, 1, 2, 3], gpu), *pools)
    assert torch.isfinite(rq[0]).all() and rq[1:].isnan().all() and rk[1:].isnan().all()
    assert pools[0][0, 1:4].isnan().all() and torch.equal(pools[1][0, :4], v.to(torch.float16))


def test_append_of_no_tokens(gpu):
    q, k, v, cos, sin = rope_inputs(gpu, 3, 2, 1, 64)
    pools = [torch.ones((2, 16, 1, 64), dtype=torch.float16, device=gpu) for _ in range(2)]
    rq, rk = ops.paged_append(q[:0], k[:0], v[:0], cos, sin, int32([], gpu), int32([], gpu), *pools)
    assert rq.shape == (0, 2, 64) and rk.shape == (0, 1, 64) and (pools[0] == 1).all()


def test_append_past_32_bits(gpu):
    """Slots whose elements lie past 2^31."""
    q, k, v, cos, sin = rope_inputs(gpu, 3, 8, 8, 128)
    pools = [torch.zeros((2100, 1024, 8, 128), dtype=torch.bfloat16, device=gpu) for _ in range(2)]
    slots = int32([2100 * 1024 - 1, 2 ** 21 + 5, 3], gpu)
    _, rk = ops.paged_append(q, k, v, cos, sin, int32([0, 1, 2], gpu), slots, *pools)
    assert torch.equal(pools[0].view(-1, 8, 128)[slots.long()], rk) and torch.equal(pools[1].view(-1, 8, 128)[slots.long()], v)
    assert int((pools[0] != 0).any(dim=(2, 3)).sum()) == 3


# ---- page copies ------------------------------------------------------------------------


@pytest.mark.parametrize("shape,moves,dtype", [((2, 8, 16, 8, 64), 1, "bf16"), ((6, 50, 64, 8, 64), 25, "fp16"),
                                               ((3, 1200, 16, 1, 8), 600, "bf16"), ((1, 9, 16, 3, 24), 4, "fp16"),
                                               ((1, 2, 128, 8, 128), 1, "bf16"), ((2, 6, 32, 5, 120), 3, "fp16")])
def test_copy_pages(gpu, shape, moves, dtype):
    pool = torch.randn(shape, device=gpu).to(DTYPES[dtype])
    order = np.random.RandomState(moves).permutation(shape[1])
    src, dst = order[:moves], order[moves:2 * moves]
    want = pool.clone()
    want[:, torch.from_numpy(dst).to(gpu)] = pool[:, torch.from_numpy(src).to(gpu)]
    ops.copy_pages(pool, src.tolist(), dst.astype(np.int32))
    assert torch.equal(pool, want)
    ops.copy_pages(pool, [], [])
    assert torch.equal(pool, want)


def test_copy_one_page_to_many_and_bits(gpu):
    """A source may serve many destinations; every bit pattern is kept."""
    pool = torch.randint(-2 ** 31, 2 ** 31 - 1, (2, 40, 16, 64), dtype=torch.int32, device=gpu)
    want = pool.clone()
    want[:, 1:31] = pool[:, :1]
    ops.copy_pages(pool, [0] * 30, range(1, 31))
    assert torch.equal(pool, want)


def test_copy_past_32_bits(gpu):
    pool = torch.zeros((3, 2100, 1024 * 1024), dtype=torch.uint8, device=gpu)
    pool[:, 2099] = torch.randint(0, 255, (3, 1024 * 1024), dtype=torch.uint8, device=gpu)
    ops.copy_pages(pool, [2099], [2098])
    assert torch.equal(pool[:, 2098], pool[:, 2099]) and not pool[:, 2097].any()


def test_append_and_copy_in_a_graph(gpu):
    """Captured together: replays take the new queries and slots, and copy what the append just stored."""
    q, k, v, cos, sin = rope_inputs(gpu, 20, 4, 2, 64, seed=3)
    pool, want = (torch.zeros((2, 400, 16, 2, 64), dtype=torch.float16, device=gpu) for _ in range(2))
    positions, slots = int32(list(range(20)), gpu), int32(list(range(20)), gpu)
    src, dst = [i % 2 for i in range(390)], list(range(10, 400))  # more moves than a launch takes

    def both(pages):
        rotated_q, _ = ops.paged_append(q, k, v, cos, sin, positions, slots, pages[0], pages[1])
        ops.copy_pages(pages, src, dst)
        return rotated_q

    both(pool)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(pool)
    for i in range(3):
        for t in (q, k, v):
            t.copy_(torch.randn_like(t))
        positions.add_(7)
        slots.copy_(torch.randperm(32, device=gpu)[:20])
        pool.zero_()
        want.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(both(want), out) and torch.equal(pool, want) and bool(pool[:, 399].any())


# ---- batch attention --------------------------------------------------------------------


def make(gpu, lengths, prefix, heads, kv, dim, dtype, page=16, seed=0, q_std=1.0, extra=0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    rng = np.random.RandomState(seed)
    held = [max(0, -(-n // page)) for n in lengths]
    prefix_pages = -(-prefix // page)
    n_pages = sum(held) + prefix_pages + 2
    order = rng.permutation(n_pages).tolist()
    width = max(held + [0]) + extra
    tables, at = [], prefix_pages
    for n in held:
        tables.append(order[at:at + n] + [-1] * (width - n))  # unused entries are never read
        at += n
    q = torch.randn((len(lengths), heads, dim), device=gpu, generator=g).mul(q_std).bfloat16()
    kp, vp = (torch.randn((n_pages, page, kv, dim), device=gpu, generator=g).to(DTYPES[dtype]) for _ in range(2))
    # what no sequence holds is NaN: reading it shows
    used = torch.zeros(n_pages * page, dtype=torch.bool)
    for i in range(prefix):
        used[order[i // page] * page + i % page] = True
    for t, n in zip(tables, lengths):
        for i in range(max(n, 0)):
            used[t[i // page] * page + i % page] = True
    for p in (kp, vp):
        p.view(-1, kv, dim)[~used.to(gpu)] = math.nan
    return q, kp, vp, tables, order[:prefix_pages]


def call(gpu, q, kp, vp, tables, lengths, prefix_table, prefix, **kw):
    width = len(tables[0]) if tables else 0
    t = torch.tensor(tables, dtype=torch.int32, device=gpu).reshape(len(tables), width)
    return ops.batch_attention(q, kp, vp, t, int32(lengths, gpu), int32(prefix_table, gpu) if prefix else None, prefix, **kw)


def check(got, q, kp, vp, tables, lengths, prefix_table, prefix, sinks=None, window=None, scale=None):
    want, size, reach = prompt.batch_attention(q, kp, vp, tables, lengths, prefix_table, prefix, sinks, window, scale)
    most = float(torch.nan_to_num(vp.double(), nan=0, posinf=0, neginf=0).abs().max())
    tol = prompt.tolerance(want, size, reach, min(prefix + max(lengths + [0]), window or 1 << 30), q.shape[2], kp.dtype,
                           torch.bfloat16, most)
    fine = torch.isfinite(want)
    got = got.double()
    assert torch.equal(torch.isfinite(got), fine)
    assert torch.equal(got[~fine].nan_to_num(nan=0.5), want[~fine].nan_to_num(nan=0.5))
    far = ((got - want).abs() / tol)[fine]
    assert far.numel() == 0 or float(far.max()) <= 1.0, float(far.max())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("heads,kv,dim", [(64, 8, 64), (8, 1, 128), (4, 4, 80), (14, 2, 8), (32, 1, 24), (6, 2, 96), (5, 5, 120)])
@pytest.mark.parametrize("lengths,prefix,window,sinks", [((1,), 0, None, True), ((40, 0, -1, 3, 129), 0, None, False),
                                                         ((1, 17, 64, -1, 0, 33), 100, None, True),
                                                         ((5, 200, 31), 70, 64, True)])
def test_batch_attention_matches_definition(gpu, dtype, heads, kv, dim, lengths, prefix, window, sinks):
    lengths = list(lengths)
    q, kp, vp, tables, pt = make(gpu, lengths, prefix, heads, kv, dim, dtype, seed=dim + prefix)
    sk = torch.randn(heads, device=gpu).bfloat16() if sinks else None
    got = call(gpu, q, kp, vp, tables, lengths, pt, prefix, sinks=sk, window=window)
    check(got, q, kp, vp, tables, lengths, pt, prefix, sk, window)
    assert not got[[i for i, n in enumerate(lengths) if n < 0]].any()


@pytest.mark.parametrize("page", [16, 32, 64, 128, 1024])
@pytest.mark.parametrize("prefix", [0, 1, 63, 64, 65, 500])
@pytest.mark.parametrize("window", [None, 1, 100])
def test_pages_and_prefixes_that_end_inside_tiles(gpu, page, prefix, window):
    lengths = [1, 32, 33, 31, 260, 64, 0, 95]
    q, kp, vp, tables, pt = make(gpu, lengths, prefix, 16, 2, 64, "fp16", page=page, seed=page + prefix, extra=3)
    got = call(gpu, q, kp, vp, tables, lengths, pt, prefix, window=window)
    check(got, q, kp, vp, tables, lengths, pt, prefix, None, window)


@pytest.mark.parametrize("count,prefix,own", [(1, 3000, 50), (2, 5000, 700), (150, 700, 30), (33, 0, 2500)])
@pytest.mark.parametrize("window", [None, 600])
def test_many_splits_and_many_sequences(gpu, count, prefix, own, window):
    rng = np.random.RandomState(count)
    lengths = [own] + rng.randint(0, own + 1, count - 1).tolist()
    q, kp, vp, tables, pt = make(gpu, lengths, prefix, 8, 1, 64, "bf16", page=64, seed=count)
    sk = torch.randn(8, device=gpu).bfloat16()
    got = call(gpu, q, kp, vp, tables, lengths, pt, prefix, window=window, sinks=sk)
    check(got, q, kp, vp, tables, lengths, pt, prefix, sk, window)


@pytest.mark.parametrize("count,prefix,heads,kv,dim,dtype,page", [
    (70, 1000, 64, 8, 64, "fp16", 64), (33, 2050, 16, 8, 64, "bf16", 16), (24, 1400, 8, 8, 128, "fp16", 32),
    (40, 1801, 20, 4, 120, "bf16", 16), (300, 1201, 32, 1, 96, "fp16", 128), (60, 8800, 4, 2, 32, "bf16", 32),
    (2, 70000, 14, 2, 128, "fp16", 16)])
def test_prefixes_read_once(gpu, count, prefix, heads, kv, dim, dtype, page):
    """Prefixes long enough for a pass of their own."""
    rng = np.random.RandomState(count)
    lengths = rng.randint(0, 150, count).tolist()
    lengths[1 % count] = -1
    q, kp, vp, tables, pt = make(gpu, lengths, prefix, heads, kv, dim, dtype, page=page, seed=count, q_std=2.0)
    q[0, 0] = 0
    q[0, 1] = 3e5  # past float16
    sk = torch.randn(heads, device=gpu).bfloat16()
    got = call(gpu, q, kp, vp, tables, lengths, pt, prefix, sinks=sk)
    check(got, q, kp, vp, tables, lengths, pt, prefix, sk)
    got = call(gpu, q, kp, vp, tables, lengths, pt[:-2] + [-5] + pt[-1:], prefix, sinks=sk)
    here = torch.tensor([n >= 0 for n in lengths], device=gpu)
    assert got[here].isnan().all() and not got[~here].any()


def test_prefix_table_within_the_tables(gpu):
    """The prefix's table may be a row of the sequences' tables."""
    q, kp, vp, tables, _ = make(gpu, [2000, 300], 0, 8, 2, 64, "fp16", seed=12)
    t, n = int32(tables, gpu), int32([1999, 300], gpu)
    for window in (None, 2500):
        got = ops.batch_attention(q, kp, vp, t, n, t[0], 1990, window=window)
        assert torch.equal(got, ops.batch_attention(q, kp, vp, t, n, t[0].clone(), 1990, window=window))
        check(got, q, kp, vp, tables, [1999, 300], tables[0], 1990, None, window)


def test_wide_tables_of_short_sequences(gpu):
    """Tables made for long sequences (many splits), sequences of a few tokens."""
    lengths = [1, 2, 40, 0]
    q, kp, vp, tables, pt = make(gpu, lengths, 30, 8, 2, 64, "fp16", extra=900)
    check(call(gpu, q, kp, vp, tables, lengths, pt, 30), q, kp, vp, tables, lengths, pt, 30)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("q_std,scale", [(40.0, None), (1e-3, None), (1e30, 1e-31), (1e-30, 1e30), (1.0, 2.0)])
def test_query_sizes(gpu, dtype, q_std, scale):
    """Queries far outside float16's range against a float16 cache, peaked and flat softmax."""
    lengths = [300, 20, 77]
    q, kp, vp, tables, pt = make(gpu, lengths, 200, 8, 2, 64, dtype, seed=3, q_std=q_std)
    q[1, 2] = 0
    sk = torch.linspace(-30, 30, 8, device=gpu).bfloat16()
    got = call(gpu, q, kp, vp, tables, lengths, pt, 200, sinks=sk, scale=scale)
    check(got, q, kp, vp, tables, lengths, pt, 200, sk, None, scale)


def test_nan_and_infinities_stay_with_their_sequence(gpu):
    lengths = [50, 60, 70]
    q, kp, vp, tables, pt = make(gpu, lengths, 40, 4, 1, 64, "fp16", seed=5)
    vp[tables[1][3], 5, 0, 9] = math.inf   # sequence 1, token 53
    vp[tables[1][3], 6, 0, 11] = math.nan
    kp[tables[2][0], 0] = math.nan
    for window in (None, 5, 30):
        got = call(gpu, q, kp, vp, tables, lengths, pt, 40, window=window)
        if window is None:
            assert got[2].isnan().all()
            check(got[:2], q[:2], kp, vp, tables[:2], lengths[:2], pt, 40)
        else:
            check(got, q, kp, vp, tables, lengths, pt, 40, None, window)


def test_bad_pages_and_lengths_make_nan(gpu):
    """Page numbers outside the pools and lengths past the table: NaN for that sequence, the others as ever."""
    lengths = [50, 60, 70, 20]
    q, kp, vp, tables, pt = make(gpu, lengths, 40, 4, 1, 64, "fp16", seed=6)
    want = call(gpu, q, kp, vp, tables, lengths, pt, 40)
    bad = [list(t) for t in tables]
    bad[1][2] = 10 ** 9
    bad[2][0] = -7
    got = call(gpu, q, kp, vp, bad, [50, 60, 70, 10 ** 6], pt, 40)
    assert torch.equal(got[0], want[0]) and got[1:].isnan().all()
    got = call(gpu, q, kp, vp, tables, lengths, [pt[0], 10 ** 6] + pt[2:], 40)
    assert got.isnan().all()
    # pages that a window has left behind are not asked for: sequence 0 sees the prefix from token 36 on, 3 from token 6
    gone = [list(t) for t in tables]
    gone[2][0] = -1
    got = call(gpu, q, kp, vp, gone, [50, 60, 70, 20], [-1] + pt[1:], 40, window=54)
    want = call(gpu, q, kp, vp, tables, lengths, pt, 40, window=54)
    assert torch.equal(got[:3], want[:3]) and torch.isfinite(got[:3]).all() and got[3].isnan().all()


def test_no_own_tables(gpu):
    """Sequences that hold the prefix alone."""
    q, kp, vp, _, pt = make(gpu, [0, 0], 90, 8, 2, 64, "bf16", seed=7)
    got = call(gpu, q, kp, vp, [[], []], [0, 0], pt, 90)
    check(got, q, kp, vp, [[], []], [0, 0], pt, 90)
    none = call(gpu, q, kp, vp, [[], []], [0, -1], [], 0)
    assert not none.any()


def test_pools_past_32_bits(gpu):
    """Pages whose elements lie past 2^31."""
    kp, vp = (torch.zeros((2100, 1024, 8, 128), dtype=torch.bfloat16, device=gpu) for _ in range(2))
    for p in (kp, vp):
        p[2097:] = torch.randn(p[2097:].shape, device=gpu)
    q = torch.randn((2, 16, 128), device=gpu).bfloat16()
    args = (q, kp, vp, [[2099], [2097]], [300, 70], [2098], 1000)
    check(call(gpu, *args), *args)


def test_streams_graphs_and_repeats(gpu):
    """The same bits on another stream and from two graphs replayed in turn with new queries."""
    lengths = [100, 400, 7]
    q, kp, vp, tables, pt = make(gpu, lengths, 300, 8, 1, 64, "fp16", seed=8)
    t, n, p = int32(tables, gpu), int32(lengths, gpu), int32(pt, gpu)
    want = ops.batch_attention(q, kp, vp, t, n, p, 300)
    torch.cuda.synchronize()
    side = torch.cuda.Stream(gpu)
    with torch.cuda.stream(side):
        other = ops.batch_attention(q, kp, vp, t, n, p, 300)
    again = ops.batch_attention(q, kp, vp, t, n, p, 300)
    torch.cuda.synchronize()
    assert torch.equal(other, want) and torch.equal(again, want)
    graphs = []
    for _ in range(2):
        out = torch.empty_like(q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.batch_attention(q, kp, vp, t, n, p, 300, out=out)
        graphs.append((graph, out))
    for i in range(4):
        q.copy_(torch.randn_like(q))
        n.copy_(int32([100 - 30 * i, 400 - i, i - 1], gpu))
        for graph, out in graphs:
            out.fill_(math.nan)
            graph.replay()
        torch.cuda.synchronize()
        want = ops.batch_attention(q, kp, vp, t, n, p, 300)
        assert all(torch.equal(out, want) for _, out in graphs)
