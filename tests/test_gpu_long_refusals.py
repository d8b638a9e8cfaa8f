"""What the operators of long conversations refuse of device tensors; no call here launches a kernel."""

from __future__ import annotations

import pytest
import torch

from klcquant_amd import ops

pytestmark = pytest.mark.gpu


def tensors(gpu):
    e = lambda *s, t=torch.bfloat16: torch.zeros(s, dtype=t, device=gpu)  # noqa: E731
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device=gpu)  # noqa: E731
    return dict(q=e(5, 8, 64), k=e(5, 2, 64), v=e(5, 2, 64), cos=e(100, 32), sin=e(100, 32), positions=i(5), slots=i(5),
                k_pages=e(4, 16, 2, 64, t=torch.float16), v_pages=e(4, 16, 2, 64, t=torch.float16), tables=i(2, 3), lengths=i(2),
                lse=e(5, 8, t=torch.float32), weights=e(3, 2, 40, t=torch.float32), rows=i(2), sinks=e(8),
                plan=ops.attention_plan([2, 3], [9, 30], 8, 2, 64), q_norm=e(64), k_norm=e(64),
                pools=e(4, 4, 16, 2, 64, t=torch.float16), layers=e(2, 3, 2, 40, t=torch.float32))


def grad(t):
    return t.clone().requires_grad_()


CHUNK = ("q", "k_pages", "v_pages", "tables", "lengths", "plan", "sinks")
WEIGHTS = ("q", "lse", "k_pages", "tables", "lengths", "plan", "weights", "rows")
EVICT = ("pools", "layers", "tables", "lengths", "rows")

SHARED = [
    ("q", lambda t: t.half(), TypeError), ("q", grad, ValueError), ("q", lambda t: t[:4], ValueError),
    ("q", lambda t: t[:, :7].contiguous(), ValueError), ("q", lambda t: t.cpu(), ValueError), ("q", lambda t: None, TypeError),
    ("q", lambda t: t.transpose(0, 1).contiguous().transpose(0, 1), ValueError), ("k_pages", lambda t: t.transpose(0, 1), ValueError),
    ("k_pages", lambda t: t.float(), TypeError), ("k_pages", grad, ValueError),
    ("k_pages", lambda t: t[..., :32].contiguous(), ValueError), ("tables", lambda t: t.long(), TypeError), ("tables", lambda t: t[:1], ValueError),
    ("tables", lambda t: t[:, ::2], ValueError), ("lengths", lambda t: t[:1], ValueError), ("lengths", lambda t: t.cpu(), ValueError),
    ("plan", lambda p: None, TypeError), ("plan", lambda p: p.data, TypeError),
    ("plan", lambda p: ops.attention_plan([5], [9], 8, 2, 64), ValueError), ("plan", lambda p: ops.attention_plan([2, 3], [9, 30], 8, 4, 64), ValueError),
    ("plan", lambda p: ops.attention_plan([2, 4], [9, 30], 8, 2, 64), ValueError)]


@pytest.mark.parametrize("name,change,error", SHARED + [
    ("v_pages", lambda t: t[:3], ValueError), ("v_pages", lambda t: t.bfloat16(), ValueError), ("sinks", lambda t: t[:7], ValueError),
    ("sinks", grad, ValueError), ("sinks", lambda t: t.float(), TypeError)])
def test_chunk_refusals(gpu, name, change, error):
    a = tensors(gpu)
    a[name] = change(a[name])
    with pytest.raises(error):
        ops.chunk_attention(*(a[n] for n in CHUNK))


def test_chunk_option_refusals(gpu):
    a = tensors(gpu)
    for kw in (dict(scale=0.0), dict(scale=float("nan")), dict(out=a["q"][:4]), dict(out=a["q"].float()), dict(out=grad(a["q"]))):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            ops.chunk_attention(*(a[n] for n in CHUNK), **kw)


@pytest.mark.parametrize("name,change,error", SHARED + [
    ("lse", lambda t: t.double(), TypeError), ("lse", lambda t: t[:4], ValueError), ("lse", lambda t: t.T.contiguous().T, ValueError),
    ("weights", lambda t: t.half(), TypeError), ("weights", lambda t: t[0], ValueError), ("weights", grad, ValueError),
    ("weights", lambda t: t[:, :1].contiguous(), ValueError), ("weights", lambda t: t[..., :0], ValueError), ("weights", lambda t: t[..., ::2], ValueError),
    ("rows", lambda t: t[:1], ValueError), ("rows", lambda t: t.long(), TypeError)])
def test_key_weight_refusals(gpu, name, change, error):
    a = tensors(gpu)
    a[name] = change(a[name])
    with pytest.raises(error):
        ops.add_key_weights(*(a[n] for n in WEIGHTS))


@pytest.mark.parametrize("name,change,error", [
    ("pools", lambda t: t.float(), TypeError), ("pools", lambda t: t[0], ValueError), ("pools", lambda t: t[:3], ValueError),
    ("pools", lambda t: t[:2], ValueError), ("pools", grad, ValueError), ("pools", lambda t: t.transpose(1, 2), ValueError),
    ("pools", lambda t: t[:, :, :8].contiguous(), ValueError), ("pools", lambda t: t.cpu(), ValueError),
    ("layers", lambda t: t.double(), TypeError), ("layers", lambda t: t[:1], ValueError), ("layers", lambda t: t[:, :, :1].contiguous(), ValueError),
    ("layers", grad, ValueError), ("layers", lambda t: t[0], ValueError), ("tables", lambda t: t.long(), TypeError), ("lengths", lambda t: t[:1], ValueError),
    ("rows", lambda t: t[:1], ValueError), ("rows", lambda t: t.cpu(), ValueError)])
def test_evict_refusals(gpu, name, change, error):
    a = tensors(gpu)
    a[name] = change(a[name])
    with pytest.raises(error):
        ops.evict_keys(*(a[n] for n in EVICT), 10)


def test_evict_option_refusals(gpu):
    a = tensors(gpu)
    for keep, kw in ((0, {}), (-1, {}), (5, dict(recent=-1)), (5, dict(first=-1)), (5, dict(recent=3, first=3)), (1 << 29, {})):
        with pytest.raises(ValueError):
            ops.evict_keys(*(a[n] for n in EVICT), keep, **kw)
    with pytest.raises(TypeError):
        ops.evict_keys(*(a[n] for n in EVICT), 5.0)


@pytest.mark.parametrize("kw,error", [
    (dict(q_norm=lambda t: t[:32]), ValueError), (dict(k_norm=lambda t: t.float()), TypeError), (dict(q_norm=grad), ValueError),
    (dict(k_norm=lambda t: t.cpu()), ValueError), (dict(q_norm=lambda t: t[None]), ValueError)])
def test_norm_refusals(gpu, kw, error):
    a = tensors(gpu)
    args = [a[n] for n in ("q", "k", "v", "cos", "sin", "positions", "slots", "k_pages", "v_pages")]
    with pytest.raises(error):
        ops.paged_append(*args, **{n: f(a[n]) for n, f in kw.items()})
    for eps in (-1e-6, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps"):
            ops.paged_append(*args, q_norm=a["q_norm"], eps=eps)
