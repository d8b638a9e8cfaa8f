"""What the operators of many sequences refuse of device tensors; no call here launches a kernel."""

from __future__ import annotations

import pytest
import torch

from klcquant_amd import ops

pytestmark = pytest.mark.gpu


def tensors(gpu):
    e = lambda *s, t=torch.bfloat16: torch.zeros(s, dtype=t, device=gpu)  # noqa: E731
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device=gpu)  # noqa: E731
    return dict(q=e(5, 8, 64), k=e(5, 2, 64), v=e(5, 2, 64), starts=i(3), sinks=e(8), cos=e(100, 32), sin=e(100, 32),
                positions=i(5), slots=i(5), k_pages=e(4, 16, 2, 64, t=torch.float16), v_pages=e(4, 16, 2, 64, t=torch.float16),
                tables=i(5, 2), lengths=i(5), prefix_table=i(2))


def grad(t):
    return t.clone().requires_grad_()


PROMPT = ("q", "k", "v", "starts", "sinks")
APPEND = ("q", "k", "v", "cos", "sin", "positions", "slots", "k_pages", "v_pages")
BATCH = ("q", "k_pages", "v_pages", "tables", "lengths", "prefix_table")


@pytest.mark.parametrize("name,change,error", [
    ("q", lambda t: t.float(), TypeError), ("k", lambda t: t.half(), TypeError), ("q", grad, ValueError),
    ("v", grad, ValueError), ("sinks", grad, ValueError), ("sinks", lambda t: t[:7], ValueError), ("sinks", lambda t: t.float(), TypeError),
    ("q", lambda t: t[:, :7].contiguous(), ValueError), ("k", lambda t: t[:4], ValueError), ("v", lambda t: t[..., :32], ValueError),
    ("q", lambda t: t.transpose(0, 1).contiguous().transpose(0, 1), ValueError), ("q", lambda t: t[..., ::2], ValueError),
    ("k", lambda t: t[:1].expand(5, 2, 64), ValueError), ("starts", lambda t: t.long(), TypeError),
    ("starts", lambda t: t[:0], ValueError), ("starts", lambda t: t.cpu(), ValueError), ("starts", lambda t: t[None], ValueError),
    ("q", lambda t: t[0], ValueError)])
def test_prompt_refusals(gpu, name, change, error):
    a = tensors(gpu)
    a[name] = change(a[name])
    with pytest.raises(error):
        ops.prompt_attention(*(a[n] for n in PROMPT))


@pytest.mark.parametrize("kw", [dict(window=0), dict(window=-4), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan"))])
def test_prompt_option_refusals(gpu, kw):
    a = tensors(gpu)
    with pytest.raises((ValueError, RuntimeError)):
        ops.prompt_attention(*(a[n] for n in PROMPT), **kw)


def test_out_refusals(gpu):
    a = tensors(gpu)
    for out in (torch.zeros(5, 8, 32, dtype=torch.bfloat16, device=gpu), a["q"].float(), a["q"].cpu(),
                torch.zeros(5, 64, 8, dtype=torch.bfloat16, device=gpu).transpose(1, 2)):
        with pytest.raises((ValueError, TypeError)):
            ops.prompt_attention(*(a[n] for n in PROMPT), out=out)
        with pytest.raises((ValueError, TypeError)):
            ops.batch_attention(*(a[n] for n in BATCH), out=out)


@pytest.mark.parametrize("name,change,error", [
    ("q", lambda t: t.half(), TypeError), ("v", grad, ValueError), ("cos", lambda t: t.float(), TypeError),
    ("sin", lambda t: t[:50], ValueError), ("cos", lambda t: t[:, :16].contiguous(), ValueError), ("positions", lambda t: t[:4], ValueError),
    ("slots", lambda t: t.long(), TypeError), ("k_pages", lambda t: t.bfloat16(), ValueError), ("v_pages", lambda t: t[:3], ValueError),
    ("k_pages", lambda t: t.float(), TypeError), ("k", lambda t: t[:, :1], ValueError), ("q", lambda t: t[..., :48].contiguous(), ValueError)])
def test_append_refusals(gpu, name, change, error):
    a = tensors(gpu)
    a[name] = change(a[name])
    with pytest.raises(error):
        ops.paged_append(*(a[n] for n in APPEND))


@pytest.mark.parametrize("name,change,error", [
    ("q", lambda t: t.half(), TypeError), ("q", grad, ValueError), ("k_pages", lambda t: t.transpose(0, 1), ValueError),
    ("v_pages", lambda t: t.bfloat16(), ValueError), ("tables", lambda t: t[:4], ValueError), ("tables", lambda t: t.long(), TypeError),
    ("tables", lambda t: t[:, ::2], ValueError), ("lengths", lambda t: t[:4], ValueError), ("lengths", lambda t: t.cpu(), ValueError),
    ("prefix_table", lambda t: t[:1], ValueError), ("prefix_table", lambda t: None, ValueError), ("q", lambda t: t[:, :7].contiguous(), ValueError)])
def test_batch_refusals(gpu, name, change, error):
    a = tensors(gpu)
    a[name] = change(a[name])
    with pytest.raises(error):
        ops.batch_attention(*(a[n] for n in BATCH), prefix_len=20)


def test_batch_option_refusals(gpu):
    a = tensors(gpu)
    for kw in (dict(prefix_len=-1), dict(prefix_len=33), dict(window=0), dict(scale=0.0)):
        with pytest.raises((ValueError, RuntimeError)):
            ops.batch_attention(*(a[n] for n in BATCH), **kw)
    odd = [torch.zeros((4, p, 2, 64), dtype=torch.float16, device=gpu) for p in (8, 24)]
    for pages in odd:
        with pytest.raises(ValueError, match="power of two"):
            ops.batch_attention(a["q"], pages, pages, a["tables"], a["lengths"])


def test_copy_refusals(gpu):
    pool = torch.zeros((2, 6, 16, 8), dtype=torch.float16, device=gpu)
    for src, dst in (([0], [6]), ([-1], [2]), ([0, 1], [2]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([3], [3]), ([[0]], [[1]])):
        with pytest.raises(ValueError):
            ops.copy_pages(pool, src, dst)
    with pytest.raises(ValueError):
        ops.copy_pages(pool.transpose(0, 1), [0], [1])
    with pytest.raises(ValueError, match="multiple of 16"):
        ops.copy_pages(torch.zeros((2, 6, 12), dtype=torch.int8, device=gpu), [0], [1])


def test_grad_and_fractions_are_refused(gpu):
    a = tensors(gpu)
    g = {n: grad(a[n]) for n in ("cos", "sin", "k_pages", "v_pages")}
    for name, t in g.items():
        with pytest.raises(ValueError, match="no backward"):
            ops.paged_append(*({**a, name: t}[n] for n in APPEND))
    for name in ("k_pages", "v_pages"):
        with pytest.raises(ValueError, match="no backward"):
            ops.batch_attention(*({**a, name: g[name]}[n] for n in BATCH), prefix_len=20)
    with pytest.raises(ValueError, match="no backward"):
        ops.copy_pages(grad(torch.zeros((2, 6, 16, 8), dtype=torch.float16, device=gpu)), [0], [1])
    with pytest.raises(ValueError, match="no backward"):
        ops.prompt_attention(*(a[n] for n in PROMPT), out=grad(a["q"]))
    with pytest.raises(TypeError):
        ops.prompt_attention(*(a[n] for n in PROMPT), window=0.5)
    with pytest.raises(TypeError):
        ops.batch_attention(*(a[n] for n in BATCH), prefix_len=2.5)
