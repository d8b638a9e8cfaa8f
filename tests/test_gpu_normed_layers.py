"""Models that normalise queries and keys, without biases: loaded from a checkpoint, and the same of both attention layers."""

from __future__ import annotations

import json
import math

import pytest
import torch

from klcquant_amd.attention import AttentionConfig, DeviceKVCache, StreamedAttention, rms_norm
from klcquant_amd.layer_tensors import LayerTensorLoader
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


@pytest.mark.parametrize("norms", ["qk", "q", "k"])
def test_streamed_layer_normalises(gpu, norms, monkeypatch):
    """A layer with norms is one without on rows whose queries and keys are normalised already."""
    config = AttentionConfig(WIDTH, HEADS, KV, DIM, rope_factor=8.0, rms_norm_eps=1e-3)
    normed, plain = layer_tensors(gpu, norms), layer_tensors(gpu, "")
    x = rows(gpu, 12, 0)
    y = x.view(12, -1, DIM).clone()
    for n, part in (("q", slice(0, HEADS)), ("k", slice(HEADS, HEADS + KV))):
        if n in norms:
            y[:, part] = rms_norm(y[:, part], normed[f"{AT}.{n}_norm.weight"], 1e-3)
    caches = [DeviceKVCache(gpu, capacity=16) for _ in range(3)]
    for p in range(12):
        got, diag = StreamedAttention(config).forward(0, x[p], normed, p, caches[0])
        with monkeypatch.context() as m:  # the path that a layer with norms takes
            m.setattr(StreamedAttention, "_step", lambda *a: None)
            want, other = StreamedAttention(config).forward(0, y[p].reshape(-1), plain, p, caches[1])
        assert torch.equal(got, want) and diag == other and got.any()
        without, _ = StreamedAttention(config).forward(0, x[p], plain, p, caches[2])
    assert not torch.equal(without, got)


def test_both_layers_give_the_same(gpu):
    """Up to roundings: the streamed layer rounds the norm's scale, its two products, the rotation's two and their sum to
    bfloat16, the batched one once, so that a query or key is off by at most 7 half steps of its size (the rotation mixes
    two elements), a score by 14 of |q| |k| / sqrt(d) and a probability by twice the most such.  Values are the same."""
    config = AttentionConfig(WIDTH, HEADS, KV, DIM, rms_norm_eps=1e-6)
    tensors = layer_tensors(gpu)
    tensors[f"{AT}.q_norm.weight"] /= 32  # scores of about one: a bound that says something
    x = rows(gpu, 20, 1)
    cache, streamed = PagedKVCache(gpu, 1, KV, DIM, 8, 16, "bf16"), DeviceKVCache(gpu, precision="bf16", capacity=32)
    a = cache.add()
    got = torch.cat([BatchedAttention(config).forward(0, x[i:i + n], tensors, cache.extend([a], n), cache)
                     for i, n in ((0, 9), (9, 5), (14, 1), (15, 5))])
    want = torch.stack([StreamedAttention(config).forward(0, x[p], tensors, p, streamed)[0] for p in range(20)])
    v = x.view(20, -1, DIM)[:, HEADS + KV:].double()
    # |x'| <= sqrt(d) max |w|, and |q| |k| / sqrt(d) <= sqrt(d) max |wq| max |wk|
    most = DIM ** 0.5 * float(tensors[f"{AT}.q_norm.weight"].abs().max()) * float(tensors[f"{AT}.k_norm.weight"].abs().max())
    score = 14 * 2.0 ** -8 * 2 ** 0.5 * most
    tol = (math.expm1(2 * score) + 4 * 2.0 ** -8) * float(v.abs().max())
    assert tol < float(want.abs().max()) and float((got.double() - want.double()).abs().max()) <= tol


def test_biases_that_are_not_there(gpu):
    config = AttentionConfig(WIDTH, HEADS, KV, DIM)
    for norms in ("", "qk"):
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


def test_the_loader_brings_them(gpu, tmp_path):
    from safetensors.torch import save_file

    held = {n: t.cpu() for n, t in layer_tensors(gpu).items()}
    other = {"model.layers.1.self_attn.q_norm.weight": torch.ones(DIM), "model.layers.1.input_layernorm.weight": torch.ones(WIDTH)}
    save_file(held | other, str(tmp_path / "model.safetensors"))
    index = {"weight_map": {n: "model.safetensors" for n in held | other}}
    (tmp_path / "model.safetensors.index.json").write_text(json.dumps(index))
    loader = LayerTensorLoader(tmp_path, gpu)
    got = loader.load(0)
    assert set(got) == set(held) and all(torch.equal(got[n].cpu(), t) for n, t in held.items())
    assert set(loader.load(1)) == set(other)
    assert set(LayerTensorLoader(tmp_path, gpu, skip=[f"{AT}.q_norm.weight"]).load(0)) == set(held) - {f"{AT}.q_norm.weight"}
