"""Rows whose visible scores are all -inf: the softmax of nothing else is NaN, as in the framework's other attention;
with a sink, or a finite score among them, they are ordinary rows.  Only a row that sees no key at all is zero."""

from __future__ import annotations

import math

import pytest
import torch

from klcquant_amd import ops

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def int32(values, gpu):
    return torch.tensor(values, dtype=torch.int32, device=gpu)


def inputs(gpu, dtype, tokens, heads, kv, dim):
    """Queries whose first element is positive, so that a key of -inf there scores -inf."""
    g = torch.Generator(device=gpu).manual_seed(dim)
    q, k, v = (torch.randn((tokens, n, dim), device=gpu, generator=g).to(DTYPES[dtype]) for n in (heads, kv, kv))
    q[..., 0] = q[..., 0].abs() + 1
    return q, k, v


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("heads,kv,dim,lengths", [(8, 2, 64, (400, 90)), (64, 64, 64, (500, 200)), (8, 2, 128, (400, 90)),
                                                  (128, 128, 128, (300, 40)), (8, 4, 40, (300, 90)), (128, 4, 64, (2101,))])
def test_prompts(gpu, dtype, heads, kv, dim, lengths):
    q, k, v = inputs(gpu, dtype, sum(lengths), heads, kv, dim)
    at = int32([0] + torch.tensor(lengths).cumsum(0).tolist(), gpu)
    clean = ops.prompt_attention(q, k, v, at)
    k[:70, ..., 0] = -math.inf  # the first sequence's first 70 keys
    k[200, ..., 0] = -math.inf
    got = ops.prompt_attention(q, k, v, at)
    assert got[:70].isnan().all() and torch.isfinite(got[70:]).all()
    assert torch.equal(got[lengths[0]:], clean[lengths[0]:])
    low = torch.full((heads,), -math.inf, dtype=torch.bfloat16, device=gpu)
    assert torch.equal(ops.prompt_attention(q, k, v, at, low).nan_to_num(nan=0.5), got.nan_to_num(nan=0.5))
    held = ops.prompt_attention(q, k, v, at, torch.zeros_like(low))
    assert not held[:70].any() and torch.isfinite(held).all()  # the sink takes all
    alone = ops.prompt_attention(q, k, v, at, window=1)
    assert alone[200].isnan().all() and torch.equal(alone[[69, 199, 201]].isnan().all(dim=2).all(dim=1).cpu(),
                                                    torch.tensor([True, False, False]))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128, 40])
@pytest.mark.parametrize("count,prefix,own", [(3, 0, 90), (3, 100, 90), (2, 3000, 700), (70, 1200, 30), (300, 64, 40)])
def test_batches(gpu, dtype, dim, count, prefix, own):
    """Sequence 0 sees -inf alone, sequence 1 one finite score, the others are not touched; no keys at all give zeros."""
    page, kv, heads = 16, 4, 8
    held, shared = -(-own // page), -(-prefix // page)
    q, k, v = inputs(gpu, dtype, (shared + count * held) * page, heads, kv, dim)
    q = q[:count].bfloat16()
    kp, vp = (x.view(-1, page, kv, dim) for x in (k, v))
    table = torch.arange(shared, dtype=torch.int32, device=gpu)
    tables = (shared + torch.arange(count * held, dtype=torch.int32, device=gpu)).view(count, held)
    lengths = int32([own] * count, gpu)
    kp[:shared, ..., 0] = -math.inf
    kp[tables[:2].flatten().long(), ..., 0] = -math.inf
    last = divmod(own - 1, page)
    kp[tables[1, last[0]].long(), last[1], :, 0] = 0
    for window in (None, own // 2):
        got = ops.batch_attention(q, kp, vp, tables, lengths, table, prefix, window=window)
        assert got[0].isnan().all() and torch.isfinite(got[1:]).all() and got[2:].any(dim=2).all()
        # sequence 1 has all its weight on its last token
        want = vp[tables[1, last[0]].long(), last[1]].float().bfloat16().repeat_interleave(heads // kv, dim=0)
        assert torch.equal(got[1], want)
        held_back = ops.batch_attention(q, kp, vp, tables, lengths, table, prefix, window=window,
                                        sinks=torch.zeros(heads, dtype=torch.bfloat16, device=gpu))
        assert not held_back[0].any() and torch.isfinite(held_back).all()
        absent = lengths.clone()
        absent[0] = -1
        for sink in (None, 0.0, math.inf, math.nan):
            sinks = None if sink is None else torch.full((heads,), sink, dtype=torch.bfloat16, device=gpu)
            assert not ops.batch_attention(q, kp, vp, tables, absent, table, prefix, sinks, window)[0].any()
    if prefix == 0:
        none = ops.batch_attention(q, kp, vp, tables, torch.zeros_like(lengths), sinks=None)
        assert not none.any()
        none = ops.batch_attention(q, kp, vp, tables, torch.zeros_like(lengths),
                                   sinks=torch.full((heads,), -math.inf, dtype=torch.bfloat16, device=gpu))
        assert not none.any()
