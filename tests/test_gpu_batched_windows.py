"""BatchedAttention's window is StreamedAttention's: 0, from the call or from the configuration, is no window."""

from __future__ import annotations

import pytest
import torch

from klcquant_amd.attention import AttentionConfig
from klcquant_amd.paged_kv import BatchedAttention, PagedKVCache

pytestmark = pytest.mark.gpu
HEADS, KV, DIM, SIZE = 8, 2, 64, 256


def layer_tensors(gpu):
    g = torch.Generator(device=gpu).manual_seed(1)
    out = {}
    for name, rows, cols in (("q", HEADS * DIM, SIZE), ("k", KV * DIM, SIZE), ("v", KV * DIM, SIZE), ("o", SIZE, HEADS * DIM)):
        at = f"model.layers.0.self_attn.{name}_proj"
        out[f"{at}.weight"] = torch.randn((rows, cols), device=gpu, generator=g).mul(cols ** -0.5).bfloat16()
        out[f"{at}.bias"] = torch.randn(rows, device=gpu, generator=g).bfloat16()
    return out


def run(gpu, configured, given):
    """A prompt and a step behind it, and the layer's output for both."""
    layer = BatchedAttention(AttentionConfig(SIZE, HEADS, KV, DIM, sliding_window=configured))
    cache = PagedKVCache(gpu, 1, KV, DIM, 8, 16)
    seqs, tensors, outs = [cache.add(), cache.add()], layer_tensors(gpu), []
    for counts in ([40, 3], [1, 2]):
        batch = cache.extend(seqs, counts)
        g = torch.Generator(device=gpu).manual_seed(batch.tokens)
        hidden = torch.randn((batch.tokens, SIZE), device=gpu, generator=g).bfloat16()
        outs.append(layer.forward(0, hidden, tensors, batch, cache, given))
    return outs


@pytest.mark.parametrize("configured,given,same", [(None, 0, None), (0, None, None), (8, 0, None), (0, 8, 8), (8, None, 8)])
def test_a_window_of_zero_is_none(gpu, configured, given, same):
    got, want = run(gpu, configured, given), run(gpu, None, same)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(got[0], run(gpu, None, None)[0]) == (same is None)
