"""What a plan asks for on the host does not go by lengths that no list is made for (no GPU)."""

from __future__ import annotations

import pytest
import torch

from klcquant_amd import ops


def test_long_sequences(monkeypatch):
    asked, empty = [], torch.empty

    def noted(size, **kw):
        asked.append(size)
        return empty(size, dtype=kw["dtype"])  # not pinned: there is no GPU

    monkeypatch.setattr(torch, "empty", noted)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    with pytest.raises(ValueError, match="too many"):  # 2^29 keys of each of 64 sequences: 134 million blocks
        ops.attention_plan([1] * 64, [(1 << 29) - 1] * 64, 8, 8, 64, key_weights=True)
    assert asked and max(asked) <= 1 << 23
    monkeypatch.setattr(torch.Tensor, "to", lambda t, *x, **kw: t)
    for key_weights in (None, False):  # attention alone
        plan = ops.attention_plan([1] * 64, [(1 << 29) - 1] * 64, 8, 8, 64, key_weights=key_weights)
        assert plan.at_list is None and plan.items >= 64
    assert ops.attention_plan([1] * 64, [100000] * 64, 8, 8, 64).list_items == 64 * 391
