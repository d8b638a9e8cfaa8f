"""Prompts whose sinks lie far above their scores: what the keys keep of the weight is as precise as without a sink
(tolerances: oracle.prompt.tolerance, relative to the rows' largest weights)."""

from __future__ import annotations

import math

import pytest
import torch

from klcquant_amd import ops
from oracle import prompt

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def make(gpu, dtype, lengths, heads, kv, dim, q_std):
    """Scores around zero, and values far enough from zero that the results stay normal numbers."""
    g = torch.Generator(device=gpu).manual_seed(heads + dim)
    tokens = sum(lengths)
    q, k, v = (torch.randn((tokens, n, dim), device=gpu, generator=g) for n in (heads, kv, kv))
    starts = torch.tensor([0] + list(lengths)).cumsum(0).tolist()
    return (q * q_std).to(dtype), k.to(dtype), (v * 100 + 2000).to(dtype), starts


def check(gpu, q, k, v, starts, sinks, window, shown=slice(None)):
    at = torch.tensor(starts, dtype=torch.int32, device=gpu)
    got = ops.prompt_attention(q, k, v, at, sinks, window)[:, shown]
    q, sinks = q[:, shown], sinks[shown]
    want, size, reach = prompt.prompt_attention(q, k, v, starts, sinks, window)
    top = prompt.largest_weights(q, k, starts, sinks, window)
    keys = min(max(b - a for a, b in zip(starts, starts[1:])), window or 1 << 30)
    most = float(torch.nan_to_num(v.double(), nan=0, posinf=0, neginf=0).abs().max())
    tol = prompt.tolerance(want, size, reach, keys, q.shape[2], q.dtype, q.dtype, most, top)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine)
    off = ((got.double() - want).abs() / tol)[fine]
    assert float(off.max()) <= 1.0, float(off.max())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("q_std", [0.0, 1.0])
@pytest.mark.parametrize("lengths,heads,kv,dim,window", [
    ((2500,), 8, 8, 64, None),         # a pair of waves for 32 rows
    ((700, 0, 33), 8, 2, 64, None),
    ((1500,), 64, 8, 64, None),        # one wave for them
    ((1100, 400), 8, 2, 64, 100),
    ((700,), 8, 2, 128, None),         # a pair of waves, and one wave
    ((900, 40), 64, 16, 128, None),
    ((600,), 8, 1, 48, 100)])
def test_sinks_above_the_scores(gpu, dtype, q_std, lengths, heads, kv, dim, window):
    """Heads with sinks 10 to 24 above scores that are all alike (0) or ordinary."""
    q, k, v, starts = make(gpu, DTYPES[dtype], lengths, heads, kv, dim, q_std)
    sinks = torch.linspace(10, 24, heads, device=gpu).bfloat16()
    check(gpu, q, k, v, starts, sinks, window)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_sinks_above_the_scores_of_many_rows(gpu, dtype):
    """Enough rows that a wave takes 64 of them."""
    q, k, v, starts = make(gpu, DTYPES[dtype], (2101,), 128, 4, 64, 1.0)
    check(gpu, q, k, v, starts, torch.linspace(8, 22, 128, device=gpu).bfloat16(), None, slice(5, 128, 31))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_sinks_above_the_scores_beside_infinities(gpu, dtype, dim):
    """Rows that are computed token by token, as a value they do not see is NaN or infinite."""
    q, k, v, starts = make(gpu, DTYPES[dtype], (700, 90), 8, 2, dim, 1.0)
    v[650, 0, 3], v[740, 1, 5] = math.nan, math.inf
    sinks = torch.linspace(10, 22, 8, device=gpu).bfloat16()
    check(gpu, q, k, v, starts, sinks, None)


def test_sinks_join_alike_in_prompts_and_batches(gpu):
    """The last token of a prompt, and the same token over pages: both within their roundings of each other."""
    n, heads, kv, dim = 2000, 8, 8, 64
    q, k, v, starts = make(gpu, torch.float16, (n,), heads, kv, dim, 1.0)
    q = q.bfloat16().half()  # the batch takes bfloat16 queries
    sinks = torch.linspace(10, 22, heads, device=gpu).bfloat16()
    last = ops.prompt_attention(q, k, v, torch.tensor(starts, dtype=torch.int32, device=gpu), sinks)[-1]
    pages = [torch.cat((x, x[:48])).view(-1, 64, kv, dim) for x in (k, v)]
    table = torch.arange(pages[0].shape[0], dtype=torch.int32, device=gpu)[None]
    step = ops.batch_attention(q[-1:].bfloat16(), *pages, table, torch.tensor([n], dtype=torch.int32, device=gpu), sinks=sinks)[0]
    # probabilities 2 x 2^-11 each, results 2^-11 and 2^-8; scores of up to 10 (the sums of |q k|), 136 2^-24 e of that
    # twice, and sums of 2,064 2^-24 twice, each: below 2^-9
    assert ((last.double() - step.double()).abs() <= last.double().abs() * (4 * 2.0 ** -11 + 2.0 ** -11 + 2.0 ** -8 + 2.0 ** -9)).all()
