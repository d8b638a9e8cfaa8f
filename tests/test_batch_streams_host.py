"""A batch's arrays and plans, made at its first layer, and layers on other streams (no GPU: streams that only take notes)."""

from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest
import torch

from klcquant_amd import ops, paged_kv
from klcquant_amd.attention import AttentionConfig

CONFIG = AttentionConfig(256, 4, 2, 64)


class Notes:
    def __init__(self):
        self.now, self.capturing, self.log = 0, False, []

    def current_stream(self, device=None):
        at = self.now
        return SimpleNamespace(record_event=lambda: self.log.append(("record", at)) or f"event of {at}",
                               wait_event=lambda e: self.log.append(("wait", at, e)))

    def tensor(self, name):
        return SimpleNamespace(record_stream=lambda stream: self.log.append(("uses", self.now, name)))


@pytest.fixture
def notes(monkeypatch):
    n = Notes()
    monkeypatch.setattr(torch.cuda, "current_stream", n.current_stream)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: n.capturing)
    monkeypatch.setattr(paged_kv, "_stream", lambda device: n.now)
    monkeypatch.setattr(paged_kv, "_to_device", lambda parts, device: tuple(n.tensor(i) for i in range(len(parts))))
    monkeypatch.setattr(ops, "attention_plan", lambda *x: SimpleNamespace(data=n.tensor(f"plan {x[5]}")))
    return n


def batch():
    on_gpu = SimpleNamespace(device=torch.device("cuda", 0), is_cuda=True)
    one = np.ones(1, np.int32)
    return paged_kv.PagedBatch(on_gpu, None, None, None, None, None, 0, False, 1, 1, dict(pages=one, keys=one, seqs=one, counts=one))


def test_other_streams_wait_for_what_the_first_layer_made(notes):
    b = batch()
    made, plan = b.sequences(), b.plan(CONFIG, None, 0)
    assert notes.log == [("record", 0)] * 2  # the default stream is one as any other
    assert b.sequences() is made and b.plan(CONFIG, None, 0) is plan and len(notes.log) == 2
    notes.now = 7
    assert b.sequences() is made
    assert notes.log[2:] == [("wait", 7, "event of 0"), ("uses", 7, 0), ("uses", 7, 1), ("uses", 7, 2)]
    del notes.log[:]
    assert b.plan(CONFIG, None, 0) is plan and notes.log == [("wait", 7, "event of 0"), ("uses", 7, "plan None")]
    del notes.log[:]
    windowed = b.plan(CONFIG, 16, 0)  # made on this one
    assert notes.log == [("record", 7)] and windowed is not plan and b.plan(CONFIG, 16, 0, False) is windowed
    notes.now = 0
    assert b.plan(CONFIG, 16, 0) is windowed and ("wait", 0, "event of 7") in notes.log


def test_a_plan_with_key_weights_does_without_them_too(notes):
    b = batch()
    both = b.plan(CONFIG, 16, 4)  # as a caller makes it before a capture
    assert b.plan(CONFIG, 16, 4, False) is both is b.plan(CONFIG, 16, 4, True)
    bare = b.plan(CONFIG, None, 0, False)
    assert b.plan(CONFIG, None, 0) is not bare


def test_a_batch_that_cannot_be_planned_stores_nothing(notes, monkeypatch):
    cache = paged_kv.PagedKVCache("cpu", 1, 2, 64, 40, 16, weighted=(2, 200))
    appended = []

    def none(*args):
        raise ValueError("too many blocks")

    monkeypatch.setattr(ops, "attention_plan", none)
    monkeypatch.setattr(ops, "paged_append", lambda *x, **kw: appended.append(x))
    at = "model.layers.0.self_attn"
    tensors = {f"{at}.{n}_proj.weight": torch.zeros(rows, 256).bfloat16() for n, rows in (("q", 256), ("k", 128), ("v", 128), ("o", 256))}
    with pytest.raises(ValueError, match="too many blocks"):
        paged_kv.BatchedAttention(CONFIG).forward(0, torch.zeros(1, 256).bfloat16(), tensors, batch(), cache)
    assert not appended


def test_a_capture_waits_for_nothing_and_makes_nothing(notes):
    b = batch()
    notes.capturing = True
    with pytest.raises(RuntimeError, match="captured"):
        b.sequences()
    notes.capturing = False
    made = b.sequences()
    notes.capturing, notes.now = True, 3
    del notes.log[:]
    assert b.sequences() is made and notes.log == []
