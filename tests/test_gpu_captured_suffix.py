"""A suffix of several tokens, captured and replayed with the next tokens' arrays copied into the batch's."""

from __future__ import annotations

import math

import pytest
import torch

from klcquant_amd.attention import AttentionConfig
from klcquant_amd.paged_kv import BatchedAttention, PagedKVCache

pytestmark = pytest.mark.gpu


def test_replays_take_the_rows_arrays(gpu, monkeypatch):
    g = torch.Generator(device=gpu).manual_seed(0)
    config = AttentionConfig(256, 4, 2, 64)
    layer, cache = BatchedAttention(config), PagedKVCache(gpu, 1, 2, 64, 20, 64)
    at = "model.layers.0.self_attn"
    tensors = {}
    for name, rows, cols in (("q_proj", 256, 256), ("k_proj", 128, 256), ("v_proj", 128, 256), ("o_proj", 256, 256)):
        tensors[f"{at}.{name}.weight"] = torch.randn((rows, cols), device=gpu, generator=g).mul_(0.05).bfloat16()
        tensors[f"{at}.{name}.bias"] = torch.zeros(rows, dtype=torch.bfloat16, device=gpu)
    seqs = [cache.add(), cache.add()]
    prompt = cache.extend(seqs, [70, 66])
    layer.forward(0, torch.randn((136, 256), device=gpu, generator=g).bfloat16(), tensors, prompt, cache)
    batch = cache.extend(seqs, 3)
    hidden = torch.randn((6, 256), device=gpu, generator=g).bfloat16()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):  # not run before: nothing of it is made on the host then
        out = layer.forward(0, hidden, tensors, batch, cache)
    graph.replay()
    for _ in range(4):
        new = cache.extend(seqs, 3)
        for name in ("positions", "slots", "lengths", "tables"):
            getattr(batch, name).copy_(getattr(new, name))
        hidden.copy_(torch.randn_like(hidden))
        out.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.isfinite(out).all()
        monkeypatch.setattr(BatchedAttention, "_suffixes", staticmethod(lambda *x: False))
        assert torch.equal(out, layer.forward(0, hidden, tensors, new, cache))
        monkeypatch.undo()
