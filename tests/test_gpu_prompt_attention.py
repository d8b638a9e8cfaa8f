"""Packed prompt attention against the float64 definition (tolerances: oracle.prompt.tolerance)."""

from __future__ import annotations

import math

import pytest
import torch

from klcquant_amd import ops
from oracle import prompt

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def make(gpu, lengths, heads, kv, dim, dtype, seed=0, q_std=1.0, fused=False, lead=0, tail=0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    tokens = lead + sum(lengths) + tail
    if fused:
        q, k, v = torch.randn((tokens, heads + 2 * kv, dim), device=gpu, generator=g).to(dtype).split((heads, kv, kv), dim=1)
    else:
        q, k, v = (torch.randn((tokens, n, dim), device=gpu, generator=g).mul(s).to(dtype)
                   for n, s in ((heads, q_std), (kv, 1.0), (kv, 1.0)))
    starts = [lead]
    for n in lengths:
        starts.append(starts[-1] + n)
    return q, k, v, starts


def device_starts(starts, gpu):
    return torch.tensor(starts, dtype=torch.int32, device=gpu)


def check(got, q, k, v, starts, sinks=None, window=None, scale=None):
    """Rows of sequences against the definition; NaN and infinities where it has them."""
    want, size, reach = prompt.prompt_attention(q, k, v, starts, sinks, window, scale)
    rows = slice(starts[0], starts[-1])
    keys = max(b - a for a, b in zip(starts, starts[1:]))
    most = float(torch.nan_to_num(v.double(), posinf=0, neginf=0).abs().max())
    tol = prompt.tolerance(want, size, reach, min(keys, window or keys), q.shape[2], q.dtype, q.dtype, most)
    got, want, tol = got.double()[rows], want[rows], tol[rows]
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine)
    assert torch.equal(got[~fine].nan_to_num(nan=0.5), want[~fine].nan_to_num(nan=0.5))
    far = ((got - want).abs() / tol)[fine]
    assert far.numel() == 0 or float(far.max()) <= 1.0, float(far.max())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("heads,kv,dim", [(8, 1, 64), (64, 8, 64), (4, 4, 128), (7, 1, 80), (16, 1, 8), (6, 2, 96),
                                          (5, 5, 24), (3, 1, 120), (40, 1, 32), (2, 1, 72), (2, 2, 16)])
@pytest.mark.parametrize("lengths,window,sinks", [((1,), None, True), ((97,), None, False), ((64, 0, 1, 200, 33), 16, True),
                                                  ((3, 130), 1, False)])
def test_prompt_attention_matches_definition(gpu, dtype, heads, kv, dim, lengths, window, sinks):
    q, k, v, starts = make(gpu, lengths, heads, kv, dim, DTYPES[dtype], seed=dim + heads)
    sk = torch.randn(heads, device=gpu).bfloat16() if sinks else None
    check(ops.prompt_attention(q, k, v, device_starts(starts, gpu), sk, window), q, k, v, starts, sk, window)


@pytest.mark.parametrize("window", [None, 1, 2, 63, 64, 65, 127, 128, 129, 500, 5000])
@pytest.mark.parametrize("dim", [64, 128])
def test_windows_across_tiles(gpu, window, dim):
    lengths = (577, 1, 64, 65, 256, 31)
    q, k, v, starts = make(gpu, lengths, 8, 2, dim, torch.bfloat16, seed=3, fused=True)
    check(ops.prompt_attention(q, k, v, device_starts(starts, gpu), None, window), q, k, v, starts, None, window)


@pytest.mark.parametrize("q_std,scale", [(30.0, None), (1.0, 3.0), (1e-3, None), (4.0, 1e-4)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_peaked_and_flat_softmax(gpu, dtype, q_std, scale):
    """Scores of hundreds (one key takes all; the running maximum moves often) and of nearly zero."""
    q, k, v, starts = make(gpu, (700, 200), 8, 1, 64, DTYPES[dtype], seed=9, q_std=q_std)
    sk = torch.linspace(-60, 60, 8, device=gpu).bfloat16()
    check(ops.prompt_attention(q, k, v, device_starts(starts, gpu), sk, None, scale), q, k, v, starts, sk, None, scale)


def test_rising_scores_move_the_maximum_every_tile(gpu):
    """Keys that grow along the sequence, so that later tiles pass the maximum by far more than 2^8."""
    q, k, v, starts = make(gpu, (600,), 4, 1, 64, torch.bfloat16, seed=2)
    q = q.abs()
    k = k.abs() * (torch.arange(600, device=gpu) / 20.0).bfloat16()[:, None, None]
    check(ops.prompt_attention(q, k, v, device_starts(starts, gpu)), q, k, v, starts)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,window", [(64, None), (64, 40), (128, None), (48, 100)])
def test_unseen_nan_and_infinities_stay_out(gpu, dtype, dim, window):
    """NaN and infinities in keys and values: rows that do not see them are as without them, rows that see them hold
    what the sum holds."""
    q, k, v, starts = make(gpu, (300, 150, 90), 8, 2, dim, DTYPES[dtype], seed=4)
    at = device_starts(starts, gpu)
    v, k = v.clone(), k.clone()
    v[200, 0, 3], v[210, 0, 3], v[233, 1, 5], v[320, 1, 0] = math.inf, -math.inf, math.nan, -math.inf
    check(ops.prompt_attention(q, k, v, at, None, window), q, k, v, starts, None, window)
    k[260:300] = math.nan  # the end of the first sequence: rows from 260 on are NaN
    k[449] = math.inf
    got = ops.prompt_attention(q, k, v, at, None, window)
    check(got, q, k, v, starts, None, window)
    assert torch.isfinite(got[:200]).all() and got[260:300].isnan().all() and torch.isfinite(got[450:]).all()


def test_infinite_values_late_in_a_long_sequence(gpu):
    q, k, v, starts = make(gpu, (1500,), 2, 1, 64, torch.bfloat16, seed=6)
    v[1499, 0, 7] = math.inf
    v[0, 0, 9] = math.nan
    check(ops.prompt_attention(q, k, v, device_starts(starts, gpu)), q, k, v, starts)


def test_sinks_at_their_limits(gpu):
    """A sink of -inf is none; one far above the scores takes all; NaN makes its head NaN."""
    q, k, v, starts = make(gpu, (100,), 4, 1, 64, torch.bfloat16, seed=7)
    at = device_starts(starts, gpu)
    bare = ops.prompt_attention(q, k, v, at)
    sk = torch.tensor([-math.inf, 3e38, math.nan, 0.5], device=gpu).bfloat16()
    got = ops.prompt_attention(q, k, v, at, sk)
    assert torch.equal(got[:, 0], bare[:, 0]) and not got[:, 1].any() and got[:, 2].isnan().all()
    check(got[:, 3:], q[:, 3:], k, v, starts, sk[3:])


def test_rows_outside_sequences_are_left(gpu):
    q, k, v, starts = make(gpu, (40, 0, 70), 8, 2, 64, torch.bfloat16, lead=37, tail=51)
    out = torch.full_like(q, 7.0)
    assert ops.prompt_attention(q, k, v, device_starts(starts, gpu), out=out) is out
    assert (out[:37] == 7).all() and (out[147:] == 7).all()
    check(out, q, k, v, starts)
    out.fill_(7.0)
    ops.prompt_attention(q, k, v, device_starts([50, 50, 50], gpu), out=out)
    assert (out == 7).all()


def test_starts_outside_the_tokens_stay_in_bounds(gpu):
    """Starts past the tokens, negative or descending: clamped, nothing outside the tensors is read or written."""
    q, k, v, _ = make(gpu, (100,), 8, 2, 64, torch.bfloat16)
    out = torch.full_like(q, 7.0)
    ops.prompt_attention(q, k, v, device_starts([-5, 40, 100000], gpu), out=out)
    check(out, q, k, v, [0, 40, 100])
    for bad in ([90, 10, 5], [100, 100, 0], [2 ** 31 - 1, -2 ** 31, 60]):
        ops.prompt_attention(q, k, v, device_starts(bad, gpu), out=out)
    torch.cuda.synchronize()


def test_many_sequences(gpu):
    """More sequences than tiles, most of one or no token."""
    lengths = [(i * 7) % 3 for i in range(1200)] + [90]
    q, k, v, starts = make(gpu, lengths, 4, 2, 64, torch.bfloat16, seed=8)
    check(ops.prompt_attention(q, k, v, device_starts(starts, gpu)), q, k, v, starts)


def test_no_tokens(gpu):
    q, k, v, _ = make(gpu, (5,), 8, 2, 64, torch.bfloat16)
    assert ops.prompt_attention(q[:0], k[:0], v[:0], device_starts([0, 0], gpu)).shape == (0, 8, 64)
    out = torch.full_like(q, 7.0)
    ops.prompt_attention(q, k, v, device_starts([0], gpu), out=out)
    assert (out == 7).all()


def test_strides_past_32_bits_of_bytes(gpu):
    """Keys and values far apart in one buffer: offsets past 2^31 elements."""
    tokens, wide = 40, 60_000_000
    flat = torch.empty(tokens * wide, dtype=torch.bfloat16, device=gpu)
    k, v = (flat.as_strided((tokens, 1, 64), (wide, 64, 1), at) for at in (0, 1024))
    k.copy_(torch.randn(k.shape, device=gpu))
    v.copy_(torch.randn(v.shape, device=gpu))
    q = torch.randn((tokens, 2, 64), device=gpu).bfloat16()
    check(ops.prompt_attention(q, k, v, device_starts([0, tokens], gpu)), q, k, v, [0, tokens])


def test_long_prompt_rows(gpu):
    """8,200 tokens: the definition at some rows (their own keys only)."""
    n, heads, dim = 8200, 8, 64
    q, k, v, _ = make(gpu, (n,), heads, 1, dim, torch.bfloat16, seed=11)
    for window in (None, 3000):
        got = ops.prompt_attention(q, k, v, device_starts([0, n], gpu), None, window)
        for row in (0, 31, 32, 2999, 3000, 4095, 8191, 8199):
            first = max(0, row - window + 1) if window else 0
            want, size, reach = prompt.attend(q[row].double(), k[first:row + 1, 0].double(), v[first:row + 1, 0].double(),
                                              torch.zeros(heads, dtype=torch.long, device=gpu),
                                              torch.full((heads,), row, device=gpu), None, dim ** -0.5)
            tol = prompt.tolerance(want, size, reach, row + 1, dim, q.dtype, q.dtype, float(v.abs().max()))
            assert ((got[row].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("lengths,heads,kv,dim,window,sinks", [((257,), 8, 2, 64, None, True), ((700,), 8, 1, 64, 256, False),
                                                               ((300, 290, 0, 530), 6, 3, 64, 270, True),
                                                               ((512,), 16, 2, 24, None, True), ((333,), 3, 1, 48, 300, False),
                                                               ((601,), 8, 2, 128, None, True), ((400, 0, 333), 3, 3, 128, 300, False),
                                                               ((450,), 6, 1, 80, None, True), ((777,), 2, 2, 104, 270, False)])
def test_few_rows_of_long_prompts(gpu, dtype, lengths, heads, kv, dim, window, sinks):
    """Few enough rows that two waves share them, and keys enough to share."""
    q, k, v, starts = make(gpu, lengths, heads, kv, dim, DTYPES[dtype], seed=dim + heads, q_std=2.0, lead=3, tail=2)
    sk = torch.randn(heads, device=gpu).bfloat16() if sinks else None
    at, out = device_starts(starts, gpu), torch.full_like(q, 7.0)
    ops.prompt_attention(q, k, v, at, sk, window, out=out)
    assert (out[:3] == 7).all() and (out[-2:] == 7).all()
    check(out, q, k, v, starts, sk, window)
    assert torch.equal(out, ops.prompt_attention(q, k, v, at, sk, window, out=torch.full_like(q, 7.0)))
    k[150], v[200, 0, 3], v[90, 0, 0] = math.nan, math.inf, -math.inf
    ops.prompt_attention(q, k, v, at, sk, window, out=out)
    check(out, q, k, v, starts, sk, window)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("lengths,dim,window,sinks", [((2101,), 64, None, True), ((2500, 0, 1900, 2200), 64, 100, False),
                                                      ((2201,), 24, None, True), ((2048,), 48, 700, False),
                                                      ((2101,), 128, None, True), ((1500, 700), 72, 500, False)])
def test_many_rows_of_long_prompts(gpu, dtype, lengths, dim, window, sinks):
    """Enough long rows that a wave takes 64 of them."""
    heads = 128
    q, k, v, starts = make(gpu, lengths, heads, 4, dim, DTYPES[dtype], seed=dim, lead=3, tail=2)
    sk = torch.randn(heads, device=gpu).bfloat16() if sinks else None
    out = torch.full_like(q, 7.0)
    ops.prompt_attention(q, k, v, device_starts(starts, gpu), sk, window, out=out)
    assert (out[:3] == 7).all() and (out[-2:] == 7).all()
    shown = slice(5, heads, 31)  # heads 5, 36, 67 and 98: one of each group
    check(out[:, shown], q[:, shown], k, v, starts, None if sk is None else sk[shown], window)
    k[400], v[1000, 2, 3], v[1500, 1, 0] = math.nan, math.inf, -math.inf
    ops.prompt_attention(q, k, v, device_starts(starts, gpu), sk, window, out=out)
    check(out[:, shown], q[:, shown], k, v, starts, None if sk is None else sk[shown], window)


def test_streams_graphs_and_repeats(gpu):
    """The same bits on another stream, twice at once, and from a graph replayed with new inputs between eager calls."""
    q, k, v, starts = make(gpu, (150, 333), 8, 2, 64, torch.bfloat16, seed=12)
    at = device_starts(starts, gpu)
    want = ops.prompt_attention(q, k, v, at)
    torch.cuda.synchronize()
    side = torch.cuda.Stream(gpu)
    with torch.cuda.stream(side):
        other = ops.prompt_attention(q, k, v, at)
    again = ops.prompt_attention(q, k, v, at)
    torch.cuda.synchronize()
    assert torch.equal(other, want) and torch.equal(again, want)
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.prompt_attention(q, k, v, at, out=out)
    for i in range(4):
        q.copy_(torch.randn_like(q))
        out.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.prompt_attention(q, k, v, at))
