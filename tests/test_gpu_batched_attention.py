"""The operators of many sequences as they are used together: BatchedAttention over a PagedKVCache, from prompts through
forks, suffixes, steps and a compaction, every row against attention's definition over its whole sequence."""

from __future__ import annotations

import math

import pytest
import torch

from klcquant_amd import ops, paged_kv
from klcquant_amd.attention import AttentionConfig
from klcquant_amd.paged_kv import BatchedAttention, PagedKVCache
from oracle import prompt

pytestmark = pytest.mark.gpu
HEADS, KV, DIM, LAYERS = 16, 8, 64, 2
WINDOWS = (None, 24)


class Run:
    """A cache, its layers and all that was put through them.  The projections select columns of the hidden rows, so
    that q, k, v and the output are exact and the comparison is of the operators alone."""

    def __init__(self, gpu, precision, page, n_pages):
        self.gpu = gpu
        width = (HEADS + 2 * KV) * DIM
        self.config = AttentionConfig(width, HEADS, KV, DIM, rope_factor=8.0)
        self.layer = BatchedAttention(self.config)
        self.cache = PagedKVCache(gpu, LAYERS, KV, DIM, n_pages, page, precision)
        self.cache.pool.fill_(math.nan)  # what is read before it is written shows
        pick = torch.eye(width, device=gpu).bfloat16()
        self.tensors = {}
        for i in range(LAYERS):
            at = f"model.layers.{i}.self_attn"
            for name, w in zip(("q_proj", "k_proj", "v_proj"), pick.split((HEADS * DIM, KV * DIM, KV * DIM))):
                self.tensors[f"{at}.{name}.weight"] = w.contiguous()
                self.tensors[f"{at}.{name}.bias"] = torch.zeros(w.shape[0], dtype=torch.bfloat16, device=gpu)
            self.tensors[f"{at}.o_proj.weight"] = pick[:, :HEADS * DIM].contiguous()
            self.tensors[f"{at}.o_proj.bias"] = torch.zeros(width, dtype=torch.bfloat16, device=gpu)
        self.tensors["model.layers.0.self_attn.sinks"] = torch.linspace(-2, 2, HEADS, device=gpu).bfloat16()
        self.rows = {}  # sequence -> its hidden rows, by layer
        self.generator = torch.Generator(device=gpu).manual_seed(page)

    def add(self):
        s = self.cache.add()
        self.rows[s] = [torch.empty((0, self.config.hidden_size), dtype=torch.bfloat16, device=self.gpu)] * LAYERS
        return s

    def fork(self, seq, count):
        children = self.cache.fork(seq, count)
        self.rows.update({c: list(self.rows[seq]) for c in children})
        return children

    def extend(self, seqs, counts, checked=None):
        before = [self.cache.length(s) for s in seqs]
        batch = self.cache.extend(seqs, counts)
        ends = [0] + torch.tensor(counts).cumsum(0).tolist()
        for i in range(LAYERS):
            hidden = torch.randn((batch.tokens, self.config.hidden_size), device=self.gpu, generator=self.generator).bfloat16()
            out = self.layer.forward(i, hidden, self.tensors, batch, self.cache, WINDOWS[i])
            assert out.shape == hidden.shape and not out[:, HEADS * DIM:].any()
            for n, s in enumerate(seqs):
                self.rows[s][i] = torch.cat((self.rows[s][i], hidden[ends[n]:ends[n + 1]]))
                if checked is None or n in checked:
                    self.check(i, s, before[n], batch.fresh, out[ends[n]:ends[n + 1], :HEADS * DIM].view(-1, HEADS, DIM))
        return batch

    def check(self, i, seq, first, fresh, got):
        """`got`: rows `first` on of the sequence in layer i.  A prompt attends to its bfloat16 keys and values, later
        tokens to the cache's, which are the float32 rotation rounded to the cache's type."""
        x = self.rows[seq][i].view(-1, HEADS + 2 * KV, DIM)
        q, k, v = (t.contiguous() for t in x.split((HEADS, KV, KV), dim=1))
        n, dtype = x.shape[0], torch.bfloat16 if fresh else self.cache.dtype
        at = torch.arange(n, dtype=torch.int32, device=self.gpu)
        cos, sin = self.layer.rope_tables(n, self.gpu)
        stored = [torch.empty((n // 16 + 1, 16, KV, DIM), dtype=self.cache.dtype, device=self.gpu) for _ in range(2)]
        q, k = ops.paged_append(q, k, v, cos, sin, at, at, *stored)
        if not fresh:
            k, v = (t.view(-1, KV, DIM)[:n] for t in stored)
        last = torch.arange(first, n, device=self.gpu)
        from_ = torch.zeros_like(last) if WINDOWS[i] is None else (last - WINDOWS[i] + 1).clamp(min=0)
        sinks = self.tensors.get(f"model.layers.{i}.self_attn.sinks")
        for h in range(HEADS):
            qh, kh, vh = q[first:, h].double(), k[:, h * KV // HEADS].double(), v[:, h * KV // HEADS].double()
            want, size, reach = prompt.attend(qh, kh, vh, from_, last, None if sinks is None else float(sinks[h]), DIM ** -0.5)
            tol = prompt.tolerance(want, size, reach, n, DIM, dtype, torch.bfloat16, float(vh.abs().max()))
            off = ((got[:, h].double() - want).abs() / tol).max()
            assert float(off) <= 1.0, (i, seq, first, h, float(off))


@pytest.mark.parametrize("precision,page", [("fp16", 16), ("bf16", 64)])
def test_prompts_forks_steps_and_compaction(gpu, precision, page):
    run = Run(gpu, precision, page, 90)
    a, b, c = run.add(), run.add(), run.add()
    batch = run.extend([a, b, c], [150, 37, 1])
    assert batch.fresh
    children = run.fork(a, 3)
    batch = run.extend(children + [b], [5, 1, 70, 2])  # a batch of several lengths, a sequence outside it
    assert not batch.fresh and batch.prefix_len == 0
    batch = run.extend(children, [1, 20, 1])
    assert batch.prefix_len == 150 // page * page
    everyone = [a, b, c] + children
    for _ in range(18):
        run.extend(everyone, [1] * 6)
    run.cache.free(b)
    run.cache.free(children[1])
    held = run.cache.compact()
    assert held == 90 - run.cache.stats()["free_pages"]
    run.cache.pool[:, held:] = math.nan
    rest = [a, c, children[0], children[2]]
    for _ in range(3):
        run.extend(rest, [1] * 4)
    d = run.add()
    run.extend([d, a], [9, 2])  # a prompt beside a suffix


def test_many_forks_of_a_long_prompt(gpu):
    """Prefixes that take a pass of their own, a suffix of several tokens and then steps."""
    run = Run(gpu, "fp16", 64, 120)
    a = run.add()
    run.extend([a], [1000])
    children = run.fork(a, 66)
    batch = run.extend(children, [2] * 66, checked=(0, 13, 65))
    assert batch.prefix_len == 960 and batch.tokens == 132
    for _ in range(2):
        run.extend(children, [1] * 66, checked=(0, 40))


def test_captured_step(gpu):
    """A decode step captured once and replayed with the next tokens' arrays copied in, against eager steps."""
    run = Run(gpu, "fp16", 64, 12)
    seqs = [run.add(), run.add()]
    run.extend(seqs, [70, 66])
    batch = run.cache.extend(seqs)
    hidden = torch.randn((2, run.config.hidden_size), device=gpu).bfloat16()
    run.layer.forward(0, hidden, run.tensors, batch, run.cache)  # the tables of RoPE, before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run.layer.forward(0, hidden, run.tensors, batch, run.cache)
    for _ in range(4):
        new = run.cache.extend(seqs)
        assert new.tables.shape == batch.tables.shape and new.prefix_len == batch.prefix_len == 0
        for name in ("positions", "slots", "lengths", "tables"):
            getattr(batch, name).copy_(getattr(new, name))
        hidden.copy_(torch.randn_like(hidden))
        out.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.isfinite(out).all()
        assert torch.equal(out, run.layer.forward(0, hidden, run.tensors, new, run.cache))


def test_more_rows_than_a_call_takes(gpu, monkeypatch):
    monkeypatch.setattr(paged_kv, "_MAX_ROWS", 7)
    run = Run(gpu, "fp16", 16, 20)
    a, b = run.add(), run.add()
    run.extend([a, b], [40, 3])
    run.extend([a, b], [18, 5])


def test_gradients_are_refused(gpu):
    run = Run(gpu, "bf16", 16, 4)
    a = run.add()
    batch = run.cache.extend([a], [3])
    hidden = torch.zeros((3, run.config.hidden_size), dtype=torch.bfloat16, device=gpu, requires_grad=True)
    with pytest.raises(ValueError, match="no backward"):
        run.layer.forward(0, hidden, run.tensors, batch, run.cache)
    with torch.no_grad():
        run.layer.forward(0, hidden, run.tensors, batch, run.cache)
