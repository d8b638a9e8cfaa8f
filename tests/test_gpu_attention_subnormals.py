"""Subnormal numbers in queries, keys, values and probabilities keep their value in the matrix instructions."""

from __future__ import annotations

import math

import pytest
import torch

from klcquant_amd import ops
from oracle import prompt

pytestmark = pytest.mark.gpu


def weigh(x: float) -> float:
    """The weight of a key that scores x beside one that scores 0."""
    return 1 / (1 + math.exp(-x))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("big,small", [(1.0, 2.0 ** -17), (1.0, 2.0 ** -20 * 1.5), (1.5, 2.0 ** -23), (3.0, 2.0 ** -22)])
def test_small_query_elements_against_float16_pages(gpu, dim, big, small):
    """Queries are scaled to float16's range by their largest element; those far below it are subnormal there."""
    q = torch.zeros((1, 2, dim), device=gpu)
    q[..., 0], q[..., 5] = big, small
    kp, vp = (torch.zeros((1, 16, 2, dim), dtype=torch.float16, device=gpu) for _ in range(2))
    kp[0, 1, :, 5] = 32768.0
    vp[0, 1] = 1.0
    scale = 0.7 / (small * 32768)  # the second key scores 0.7
    got = ops.batch_attention(q.bfloat16(), kp, vp, torch.zeros((1, 1), dtype=torch.int32, device=gpu),
                              torch.tensor([2], dtype=torch.int32, device=gpu), scale=scale)
    # the element may be off by 2^-25 of the largest, the probabilities and the result by 2^-11 and 2^-8
    off = 0.7 * 2.0 ** -25 * big / small
    assert (got.double() - weigh(0.7)).abs().max() <= off + 2.0 ** -10 + 2.0 ** -8


@pytest.mark.parametrize("dim", [64, 128, 40])
def test_subnormal_float16_prompts(gpu, dim):
    """Elements of 2^-20 in float16 queries, keys and values."""
    tiny = 2.0 ** -20
    q, k, v = (torch.zeros((300, n, dim), dtype=torch.float16, device=gpu) for n in (4, 2, 2))
    starts = torch.tensor([0, 300], dtype=torch.int32, device=gpu)
    v[:] = 48 * tiny
    assert torch.equal(ops.prompt_attention(q, k, v, starts), v.repeat_interleave(2, dim=1))
    q[..., 1], k[0, :, 1], v[:] = tiny, 1024.0, 0
    v[0] = 1.0
    for a, b in ((q, k), (k, q)):  # subnormal queries, then subnormal keys
        q2, k2 = (q, k) if a is q else (torch.zeros_like(q), torch.zeros_like(k))
        if a is k:
            q2[..., 1], k2[0, :, 1] = 1024.0, tiny
        got = ops.prompt_attention(q2, k2, v, starts, scale=3.0 / (tiny * 1024)).double()
        n = torch.arange(300, device=gpu, dtype=torch.float64)[:, None, None]
        want = math.exp(3) / (math.exp(3) + n)
        assert ((got - want).abs() <= want * (2 * 2.0 ** -11 + 2.0 ** -11 + 2.0 ** -16)).all()


def test_subnormal_probabilities_in_float16(gpu):
    """8,000 keys whose probabilities are 2^-16 of the largest one's: float16 holds them as subnormals."""
    n, dim = 8000, 64
    q, k, v = (torch.zeros((n, 1, dim), dtype=torch.float16, device=gpu) for _ in range(3))
    q[..., 0], k[0, :, 0], v[1:] = 1.0, 1.0, 8.0
    got = ops.prompt_attention(q, k, v, torch.tensor([0, n], dtype=torch.int32, device=gpu), scale=16 * math.log(2)).double()
    share = torch.arange(n, device=gpu, dtype=torch.float64)[:, None, None] * 2.0 ** -16
    want = 8 * share / (1 + share)
    assert ((got - want).abs() <= want * (2.0 ** -8 + 2 * 2.0 ** -11) + 2.0 ** -25).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_subnormal_bfloat16_values(gpu, dim):
    """bfloat16 values below 2^-126, alike for all keys: the result is that value."""
    q, k = (torch.randn((200, n, dim), device=gpu).bfloat16() for n in (4, 2))
    v = torch.full((200, 2, dim), 2.0 ** -130, device=gpu).bfloat16()
    assert float(v.double().max()) == 2.0 ** -130
    got = ops.prompt_attention(q, k, v, torch.tensor([0, 200], dtype=torch.int32, device=gpu)).double()
    assert ((got - 2.0 ** -130).abs() <= 2.0 ** -133).all()
