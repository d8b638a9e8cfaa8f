"""Normed append, chunk attention, key weights and eviction as they are used together: BatchedAttention over a cache that
keeps weights, from prompts through forks, suffixes, evictions, steps and a compaction, every row against attention's
definition over the keys that its head still holds."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from klcquant_amd import ops
from klcquant_amd.attention import AttentionConfig
from klcquant_amd.paged_kv import BatchedAttention, PagedKVCache
from oracle import chunk, prompt

pytestmark = pytest.mark.gpu
HEADS, KV, DIM, LAYERS = 8, 4, 64, 2
WINDOWS = (None, 24)


class Run:
    """A cache, its layers, and a model of what each head of each layer holds.  The projections select columns of the
    hidden rows, so that q, k, v and the output are exact and the comparison is of the operators alone."""

    def __init__(self, gpu, precision, page, n_pages, first_tokens=0, weighted=(8, 400), norms=True):
        self.gpu, self.first = gpu, first_tokens
        width = (HEADS + 2 * KV) * DIM
        self.config = AttentionConfig(width, HEADS, KV, DIM, rope_factor=8.0)
        self.layer = BatchedAttention(self.config, first_tokens)
        self.cache = PagedKVCache(gpu, LAYERS, KV, DIM, n_pages, page, precision, weighted)
        self.cache.pool.fill_(math.nan)  # what is read before it is written shows
        if weighted:
            self.cache.weights.fill_(math.nan)
        pick = torch.eye(width, device=gpu).bfloat16()
        self.tensors = {}
        for i in range(LAYERS):
            at = f"model.layers.{i}.self_attn"
            for name, w in zip(("q_proj", "k_proj", "v_proj"), pick.split((HEADS * DIM, KV * DIM, KV * DIM))):
                self.tensors[f"{at}.{name}.weight"] = w.contiguous()
                self.tensors[f"{at}.{name}.bias"] = torch.zeros(w.shape[0], dtype=torch.bfloat16, device=gpu)
            self.tensors[f"{at}.o_proj.weight"] = pick[:, :HEADS * DIM].contiguous()
            self.tensors[f"{at}.o_proj.bias"] = torch.zeros(width, dtype=torch.bfloat16, device=gpu)
        if norms:
            self.tensors["model.layers.0.self_attn.q_norm.weight"] = torch.linspace(0.5, 2, DIM, device=gpu).bfloat16()
            self.tensors["model.layers.0.self_attn.k_norm.weight"] = torch.linspace(1.5, 0.7, DIM, device=gpu).bfloat16()
        self.tensors["model.layers.1.self_attn.sinks"] = torch.linspace(-2, 2, HEADS, device=gpu).bfloat16()
        self.held = {}   # sequence -> layer -> [keys, values, weights] of [n, KV, ...]
        self.seen = {}   # sequence -> tokens so far
        self.generator = torch.Generator(device=gpu).manual_seed(page)

    def add(self):
        s = self.cache.add()
        empty = lambda *x: torch.zeros((0, KV, *x), dtype=torch.float64, device=self.gpu)  # noqa: E731
        self.held[s] = [[empty(DIM), empty(DIM), empty()] for _ in range(LAYERS)]
        self.seen[s] = 0
        return s

    def fork(self, seq, count):
        children = self.cache.fork(seq, count)
        for c in children:
            self.held[c] = [[t.clone() for t in layer] for layer in self.held[seq]]
            self.seen[c] = self.seen[seq]
        return children

    def extend(self, seqs, counts):
        batch = self.cache.extend(seqs, counts)
        assert batch.positions.tolist() == [self.seen[s] + i for s, n in zip(seqs, counts) for i in range(n)]
        ends = np.concatenate(([0], np.cumsum(counts)))
        for i in range(LAYERS):
            hidden = torch.randn((batch.tokens, self.config.hidden_size), device=self.gpu, generator=self.generator).bfloat16()
            out = self.layer.forward(i, hidden, self.tensors, batch, self.cache, WINDOWS[i])
            assert out.shape == hidden.shape and not out[:, HEADS * DIM:].any()
            at = f"model.layers.{i}.self_attn"
            q, k, v = (t.contiguous() for t in hidden.view(-1, HEADS + 2 * KV, DIM).split((HEADS, KV, KV), dim=1))
            stored = [torch.empty((batch.tokens // 16 + 1, 16, KV, DIM), dtype=self.cache.dtype, device=self.gpu) for _ in range(2)]
            cos, sin = self.layer.rope_tables(batch.end, self.gpu)
            slots = torch.arange(batch.tokens, dtype=torch.int32, device=self.gpu)
            q, _ = ops.paged_append(q, k, v, cos, sin, batch.positions, slots, *stored, q_norm=self.tensors.get(f"{at}.q_norm.weight"),
                                    k_norm=self.tensors.get(f"{at}.k_norm.weight"), eps=self.config.rms_norm_eps)
            k, v = (t.view(-1, KV, DIM) for t in stored)
            for n, s in enumerate(seqs):
                rows = slice(int(ends[n]), int(ends[n + 1]))
                self.check(i, s, q[rows], k[rows], v[rows], out[rows, :HEADS * DIM].view(-1, HEADS, DIM))
        for s, n in zip(seqs, counts):
            self.seen[s] += n
        return batch

    def check(self, i, seq, q, k, v, got):
        held = self.held[seq][i]
        held[0], held[1] = torch.cat((held[0], k.double())), torch.cat((held[1], v.double()))
        n = held[0].shape[0]
        rows = torch.arange(n - q.shape[0], n, device=self.gpu)
        sinks = self.tensors.get(f"model.layers.{i}.self_attn.sinks")
        want, _, w, size, reach = chunk.attend(q, held[0], held[1], rows, sinks, WINDOWS[i], self.first if WINDOWS[i] else 0, DIM ** -0.5)
        tol = prompt.tolerance(want, size, reach, n, DIM, self.cache.dtype, torch.bfloat16, float(held[1].abs().max()))
        # a layer without weights takes whole prompts' bfloat16 keys and values
        assert float(((got.double() - want).abs() / tol).max()) <= 1.0, (i, seq, float(((got.double() - want).abs() / tol).max()))
        if self.cache.weights is None:
            return
        new = w.view(q.shape[0], KV, HEADS // KV, n).sum(dim=(0, 2)).T
        held[2] = torch.cat((held[2], torch.zeros((q.shape[0], KV), dtype=torch.float64, device=self.gpu))) + new
        weights = self.cache.weights[i, seq, :, :n].T.double()
        assert torch.allclose(weights, held[2], rtol=2e-4, atol=1e-30), (i, seq, float((weights - held[2]).abs().max()))

    def evict(self, seqs, keep, recent, first):
        before = self.cache.weights.cpu().numpy()
        cut = [s for s in seqs if self.cache.length(s) > keep]
        assert self.cache.evict(seqs, keep, recent, first) == cut
        for s in cut:
            assert self.cache.length(s) == keep
            for i in range(LAYERS):
                held = self.held[s][i]
                n = held[0].shape[0]
                old = torch.stack([torch.from_numpy(chunk.kept_places(before[i, s, h], n, keep, recent, first))
                                   for h in range(KV)], dim=1).to(self.gpu)
                self.held[s][i] = [torch.gather(t, 0, old.view(keep, KV, *[1] * (t.dim() - 2)).expand(keep, *t.shape[1:])) for t in held]


@pytest.mark.parametrize("precision,page", [("fp16", 16), ("bf16", 64)])
def test_prompts_forks_suffixes_evictions_and_steps(gpu, precision, page):
    run = Run(gpu, precision, page, 60)
    a, b, c = run.add(), run.add(), run.add()
    assert run.extend([a, b, c], [150, 37, 1]).fresh
    children = run.fork(a, 2)
    run.extend(children + [b], [5, 1, 70])
    free = run.cache.stats()["free_pages"]
    run.evict([a, b, children[0]], 96, 24, 4)  # shared pages are copied first: the other child keeps its own
    assert run.cache.stats()["free_pages"] != free
    run.extend([a, b, c, *children], [1, 30, 2, 1, 9])
    for _ in range(4):
        run.extend([a, b, c, *children], [1] * 5)
    run.evict([a, b, c, *children], 96, 24, 4)
    child, = run.fork(a, 1)
    run.extend([child, a], [3, 1])
    run.cache.free(b)
    held = run.cache.compact()
    run.cache.pool[:, held:] = math.nan
    for _ in range(3):
        run.extend([a, c, child, *children], [1] * 5)
    d = run.add()
    run.extend([d, a], [19, 2])  # a prompt beside a suffix
    run.evict([d], 19, 24 - 5, 0)
    run.evict([d], 18, 0, 0)


@pytest.mark.parametrize("first", [1, 5, 40])
def test_first_tokens_beside_windows(gpu, first):
    """Without weights: prompts, suffixes and steps of the windowed layer see its first tokens too."""
    run = Run(gpu, "bf16", 16, 60, first_tokens=first, weighted=None, norms=False)
    a, b = run.add(), run.add()
    run.extend([a, b], [200, 3])
    run.extend([a, b], [7, 60])
    for _ in range(3):
        run.extend([a, b], [1, 1])


def test_a_cache_stays_within_its_keys(gpu):
    """A conversation longer than the cache could hold: cut whenever it is full."""
    run = Run(gpu, "fp16", 16, 9, weighted=(1, 144))
    a = run.add()
    run.extend([a], [100])
    for i in range(12):
        run.extend([a], [11 + i])
        run.evict([a], 100, 30, 2)
    assert run.seen[a] == 100 + sum(range(11, 23)) and run.cache.length(a) == 100
    with pytest.raises(RuntimeError, match="weights of 144 keys"):
        run.cache.extend([a], [45])
    assert run.cache.length(a) == 100
    with pytest.raises(RuntimeError, match="1 sequences"):
        run.cache.add()
    with pytest.raises(RuntimeError, match="1 sequences"):
        run.cache.fork(a)
    assert run.cache.stats()["sequences"] == 1
    run.extend([a], [44])


def test_captured_step_of_a_weighted_cache(gpu):
    """A step captured once and replayed with the next tokens' arrays copied in, against eager steps of a twin."""
    runs = [Run(gpu, "fp16", 64, 12) for _ in range(2)]
    for run in runs:
        run.generator.manual_seed(1)
        assert [run.add(), run.add()] == [0, 1]
        run.extend([0, 1], [70, 66])
    run, twin = runs
    batch, other = run.cache.extend([0, 1]), twin.cache.extend([0, 1])
    hidden = torch.randn((2, run.config.hidden_size), device=gpu).bfloat16()
    run.layer.forward(0, hidden, run.tensors, batch, run.cache, 0)
    twin.layer.forward(0, hidden, twin.tensors, other, twin.cache, 0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run.layer.forward(0, hidden, run.tensors, batch, run.cache, 0)
    for _ in range(4):
        new, other = run.cache.extend([0, 1]), twin.cache.extend([0, 1])
        for name in ("positions", "slots"):
            getattr(batch, name).copy_(getattr(new, name))
        for mine, theirs in zip(batch.sequences(), new.sequences()):
            mine.copy_(theirs)
        hidden.copy_(torch.randn_like(hidden))
        graph.replay()
        torch.cuda.synchronize()
        want = twin.layer.forward(0, hidden, twin.tensors, other, twin.cache, 0)
        assert torch.equal(out, want)
        assert torch.equal(run.cache.weights.nan_to_num(nan=-1.0)[0], twin.cache.weights.nan_to_num(nan=-1.0)[0])
    fresh = run.cache.extend([0, 1])
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            run.layer.forward(0, hidden, run.tensors, fresh, run.cache, 0)


def test_gradients_are_refused(gpu):
    run = Run(gpu, "bf16", 16, 8)
    a = run.add()
    batch = run.cache.extend([a], [3])
    hidden = torch.zeros((3, run.config.hidden_size), dtype=torch.bfloat16, device=gpu, requires_grad=True)
    with pytest.raises(ValueError, match="no backward"):
        run.layer.forward(0, hidden, run.tensors, batch, run.cache)
