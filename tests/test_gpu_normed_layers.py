"""Models that normalise queries and keys, without biases."""

from __future__ import annotations

import pytest
import torch

from klcquant_amd.attention import AttentionConfig, DeviceKVCache, StreamedAttention
from klcquant_amd.paged_kv import BatchedAttention, PagedKVCache

pytestmark = pytest.mark.gpu
HEADS, KV, DIM = 8, 2, 64
WIDTH = (HEADS + 2 * KV) * DIM
AT = "model.layers.0.self_attn"


def layer_tensors(gpu, norms=("q", "k")):
    """Projections that select columns of the hidden row, so that q, k, v and the output are exact."""
    pick = torch.eye(WIDTH, device=gpu).bfloat16()
    t = {f"{AT}.{n}_proj.weight": w.contiguous() for n, w in zip("qkv", pick.split((HEADS * DIM, KV * DIM, KV * DIM)))}
    t[f"{AT}.o_proj.weight"] = pick[:, :HEADS * DIM].contiguous()
    t |= {f"{AT}.{n}_norm.weight": torch.linspace(0.4, 1.8 + (n == "k"), DIM, device=gpu).bfloat16() for n in norms}
    return t


def rows(gpu, n, seed):
    g = torch.Generator(device=gpu).manual_seed(seed)
    return torch.randn((n, WIDTH), device=gpu, generator=g).mul_(3.0).bfloat16()


def test_biases_that_are_not_there(gpu):
    config = AttentionConfig(WIDTH, HEADS, KV, DIM)
    for norms in ("",):
        bare = layer_tensors(gpu, norms)
        zero = bare | {f"{AT}.{n}_proj.bias": torch.zeros(bare[f"{AT}.{n}_proj.weight"].shape[0], dtype=torch.bfloat16, device=gpu)
                       for n in "qkvo"}
        x, outs = rows(gpu, 5, 2), []
        for tensors in (bare, zero):
            cache = PagedKVCache(gpu, 1, KV, DIM, 8, 16)
            streamed = DeviceKVCache(gpu, capacity=8)
            outs.append((BatchedAttention(config).forward(0, x, tensors, cache.extend([cache.add()], 5), cache),
                         StreamedAttention(config).forward(0, x[0], tensors, 0, streamed)[0]))
        assert torch.equal(outs[0][0], outs[1][0])
        # one token's context is its value, rounded once, on every path
        assert torch.equal(outs[0][1], outs[1][1])
