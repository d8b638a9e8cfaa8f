"""Layers of one batch on several streams: the first makes the batch's arrays and plans, the others wait for them."""

from __future__ import annotations

import math

import pytest
import torch

from klcquant_amd.attention import AttentionConfig
from klcquant_amd.paged_kv import BatchedAttention, PagedKVCache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("weighted", [None, (3, 200)])
def test_a_layer_beside_the_first(gpu, weighted):
    g = torch.Generator(device=gpu).manual_seed(0)
    config = AttentionConfig(256, 4, 2, 64)
    layer, cache = BatchedAttention(config), PagedKVCache(gpu, 2, 2, 64, 20, 64, weighted=weighted)
    tensors = {}
    for i in range(2):
        for name, rows in (("q_proj", 256), ("k_proj", 128), ("v_proj", 128), ("o_proj", 256)):
            at = f"model.layers.{i}.self_attn.{name}"
            tensors[f"{at}.weight"] = torch.randn((rows, 256), device=gpu, generator=g).mul_(0.05).bfloat16()
            tensors[f"{at}.bias"] = torch.zeros(rows, dtype=torch.bfloat16, device=gpu)
    cache.pool.zero_()
    seqs = [cache.add(), cache.add()]
    prompt = cache.extend(seqs, [70, 66])
    start = torch.randn((136, 256), device=gpu, generator=g).bfloat16()
    for i in range(2):
        layer.forward(i, start, tensors, prompt, cache)
    hidden = torch.randn((6, 256), device=gpu, generator=g).bfloat16()
    streams = [torch.cuda.Stream(gpu) for _ in range(2)]
    kept = cache.pool.clone(), None if weighted is None else cache.weights.clone()

    def run(side_by_side):
        cache.pool.copy_(kept[0])
        if weighted is not None:
            cache.weights.copy_(kept[1])
        batch = cache.extend(seqs, 3)
        torch.cuda.synchronize()
        outs = []
        for i in range(2):
            with torch.cuda.stream(streams[i if side_by_side else 0]):
                if side_by_side and i == 0:
                    torch.cuda._sleep(20_000_000)  # the arrays' copies come late
                outs.append(layer.forward(i, hidden, tensors, batch, cache))
        torch.cuda.synchronize()
        cache.table.undo_extend(seqs, [3, 3])
        return outs

    want = run(False)
    for _ in range(3):
        got = run(True)
        assert all(torch.equal(a, b) and torch.isfinite(a).all() for a, b in zip(got, want))
    assert math.isfinite(float(cache.pool.float().sum()))


def test_a_step_captured_without_a_run(gpu):
    """A weighted cache's step, captured once its arrays and plans are made and never run before: each replay adds its
    tokens' weights once, as eager steps of a twin do."""
    from test_gpu_long_conversations import WINDOWS, Run

    runs = [Run(gpu, "fp16", 64, 12, first_tokens=3) for _ in range(2)]
    for run in runs:
        run.generator.manual_seed(1)
        assert [run.add(), run.add()] == [0, 1]
        run.extend([0, 1], [70, 66])
    run, twin = runs
    batch, other = run.cache.extend([0, 1]), twin.cache.extend([0, 1])
    hidden = torch.randn((2, run.config.hidden_size), device=gpu).bfloat16()
    batch.sequences()
    for window in WINDOWS:
        batch.plan(run.config, window, 3 if window else 0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [run.layer.forward(i, hidden, run.tensors, batch, run.cache, WINDOWS[i]) for i in range(2)]
    for step in range(4):
        if step:
            new, other = run.cache.extend([0, 1]), twin.cache.extend([0, 1])
            for name in ("positions", "slots"):
                getattr(batch, name).copy_(getattr(new, name))
            for mine, theirs in zip(batch.sequences(), new.sequences()):
                mine.copy_(theirs)
            hidden.copy_(torch.randn_like(hidden))
        graph.replay()
        torch.cuda.synchronize()
        want = [twin.layer.forward(i, hidden, twin.tensors, other, twin.cache, WINDOWS[i]) for i in range(2)]
        assert all(torch.equal(a, b) and torch.isfinite(a).all() for a, b in zip(outs, want))
        assert torch.equal(run.cache.weights.nan_to_num(nan=-1.0), twin.cache.weights.nan_to_num(nan=-1.0))
