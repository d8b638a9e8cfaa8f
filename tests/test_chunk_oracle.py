"""The definitions of chunk attention and eviction on small cases that can be worked out by hand (no GPU)."""

from __future__ import annotations

import math

import numpy as np
import torch

from oracle import chunk


def test_what_a_token_sees():
    rows, keys = torch.tensor([-1, 0, 5]), torch.arange(7)
    assert chunk.sees(rows, keys, None, 0).sum(dim=1).tolist() == [0, 1, 6]
    assert chunk.sees(rows, keys, 2, 0)[2].nonzero().flatten().tolist() == [4, 5]
    assert chunk.sees(rows, keys, 2, 2)[2].nonzero().flatten().tolist() == [0, 1, 4, 5]
    assert chunk.sees(rows, keys, 2, 9)[2].nonzero().flatten().tolist() == [0, 1, 2, 3, 4, 5]


def test_attention_of_equal_scores():
    q, k = torch.zeros(2, 2, 8), torch.ones(3, 1, 8, dtype=torch.float64)
    v = torch.arange(3.0, dtype=torch.float64).view(3, 1, 1).expand(3, 1, 8)
    out, lse, w, _, _ = chunk.attend(q, k, v, torch.tensor([1, 2]), None, None, 0, 1.0)
    assert torch.allclose(out[:, 0, 0], torch.tensor([0.5, 1.0], dtype=torch.float64))
    assert torch.allclose(lse[:, 1], torch.tensor([math.log(2), math.log(3)], dtype=torch.float64))
    assert torch.allclose(w.sum(dim=2), torch.ones(2, 2, dtype=torch.float64))
    out, lse, _, _, _ = chunk.attend(q, k, v, torch.tensor([-1, 2]), torch.zeros(2), None, 0, 1.0)
    assert not out[0].any() and lse[0].tolist() == [0, 0] and torch.allclose(lse[1].exp(), torch.full((2,), 4.0, dtype=torch.float64))
    out, lse, _, _, _ = chunk.attend(q, k, v, torch.tensor([-1, 2]), None, None, 0, 1.0)
    assert not out[0].any() and (lse[0] == -math.inf).all()


def test_which_keys_stay():
    w = np.array([0, 5, 1, 3, 3, 2, 9, 0], np.float32)
    assert chunk.kept_places(w, 8, 8, 2, 1).tolist() == list(range(8))
    assert chunk.kept_places(w, 3, 5, 1, 0).tolist() == [0, 1, 2, -1, -1]
    # the first, the last two, and of the middle 5 and the earlier 3: place 2 is free and takes key 3
    assert chunk.kept_places(w, 8, 5, 2, 1).tolist() == [0, 1, 3, 6, 7]
    # no first ones: 5, 3, 3 stay
    assert chunk.kept_places(w, 8, 5, 2, 0).tolist() == [3, 1, 4, 6, 7]
    assert chunk.kept_places(w, 8, 3, 2, 1).tolist() == [0, 6, 7]
    w[2] = math.nan
    w[4] = math.inf
    assert chunk.kept_places(w, 8, 4, 2, 0).tolist() == [2, 4, 6, 7]
