"""oracle/prompt.py against closed forms and the decode oracle."""

from __future__ import annotations

import math

import numpy as np
import torch

from oracle import attention as oat
from oracle import prompt
from oracle.numerics import bf16_to_f32, f32_to_bf16


def test_one_key_and_a_sink():
    """One key of score s and a sink of logit t: the key's weight is 1 / (1 + exp(t - s))."""
    q = torch.tensor([[[2.0, 0.0]]])
    k = torch.tensor([[[3.0, 1.0]]])
    v = torch.tensor([[[5.0, -7.0]]])
    out, size, _ = prompt.prompt_attention(q, k, v, [0, 1], sinks=torch.tensor([1.5]), scale=0.5)
    w = 1 / (1 + math.exp(1.5 - 3.0))
    assert torch.allclose(out[0, 0], w * torch.tensor([5.0, -7.0], dtype=torch.float64), rtol=1e-14)
    assert torch.allclose(size[0, 0], w * torch.tensor([5.0, 7.0], dtype=torch.float64), rtol=1e-14)


def test_equal_keys_average_the_window():
    """Keys that all score alike: row i is the mean of the values it sees."""
    v = torch.arange(12.0).reshape(12, 1, 1)
    q, k = torch.ones(12, 1, 1), torch.ones(12, 1, 1)
    out, _, _ = prompt.prompt_attention(q, k, v, [0, 5, 5, 12], window=3)
    want = [0, 0.5, 1, 2, 3, 5, 5.5, 6, 7, 8, 9, 10]
    assert torch.allclose(out[:, 0, 0], torch.tensor(want, dtype=torch.float64))


def test_unseen_nan_and_infinities_stay_out():
    v = torch.tensor([1.0, 2.0, math.inf, math.nan]).reshape(4, 1, 1)
    out, _, _ = prompt.prompt_attention(torch.ones(4, 1, 1), torch.ones(4, 1, 1), v, [0, 4])
    assert out[:2, 0, 0].tolist() == [1.0, 1.5] and out[2, 0, 0] == math.inf and out[3, 0, 0].isnan()


def test_last_row_is_the_decode_oracles_context():
    """The prompt's last row, and the batch's row over pages, against the decode oracle (which rounds probabilities)."""
    rng = np.random.default_rng(5)
    n, heads, kv, dim, page = 70, 4, 2, 16, 16
    q, k, v = (f32_to_bf16(rng.standard_normal(s).astype(np.float32)) for s in ((n, heads, dim), (n, kv, dim), (n, kv, dim)))
    sinks = f32_to_bf16(rng.standard_normal(heads).astype(np.float32))
    t = lambda x: torch.from_numpy(bf16_to_f32(x))  # noqa: E731
    for window in (None, 33):
        want = bf16_to_f32(oat.decode_attention(q[-1], k, v, sinks, window=window)[0])
        out, size, _ = prompt.prompt_attention(t(q), t(k), t(v), [0, n], t(sinks), window)
        off = 2.0 ** -8 * (size[-1] + 2 * out[-1].abs()) + 1e-6  # probabilities, context twice
        assert ((out[-1] - torch.from_numpy(want)).abs() <= off).all()
        order = rng.permutation(8)
        kp, vp = np.zeros((8, page, kv, dim), np.float32), np.zeros((8, page, kv, dim), np.float32)
        for i in range(n):  # the first 20 tokens are the prefix, in pages of its own
            at = (order[i // page], i % page) if i < 20 else (order[2 + (i - 20) // page], (i - 20) % page)
            kp[at], vp[at] = bf16_to_f32(k[i]), bf16_to_f32(v[i])
        got, _, _ = prompt.batch_attention(t(q)[-1:], torch.from_numpy(kp), torch.from_numpy(vp), [order[2:].tolist()],
                                           [n - 20], order[:2].tolist(), 20, t(sinks), window)
        assert torch.allclose(got[0], out[-1], rtol=1e-12, atol=1e-12)
