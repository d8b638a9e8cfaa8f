"""Attention of packed prompts and of a decode batch, in float64 (test infrastructure only).

``attend`` is the definition, one head of one sequence at a time: softmax of
``scale * q . k`` over the keys that a row sees, and the sink logit, which has
no value; a row that sees no key is zero (with a sink of -inf too, which is
none), one that sees keys whose scores are all -inf is NaN.  Values that a row
does not see do not enter its sum, whatever they hold.
"""

from __future__ import annotations

import math

import torch


def weights(q: torch.Tensor, k: torch.Tensor, first: torch.Tensor, last: torch.Tensor, sink: float | None,
            scale: float) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys' weights ``[R, N]`` of float64 ``q [R, D]`` and ``k [N, D]``, and which keys a row sees:
    ``first[r]..last[r]`` (none if last < first)."""
    n = k.shape[0]
    at = torch.arange(n, device=q.device)
    seen = (at[None, :] >= first[:, None]) & (at[None, :] <= last[:, None])
    score = torch.where(seen, q @ k.T.contiguous() * scale, -math.inf)
    top = score.amax(dim=1, keepdim=True) if n else torch.full((q.shape[0], 1), -math.inf, dtype=torch.float64, device=q.device)
    if sink is not None:
        top = torch.clamp(top, min=sink)
    base = torch.where(torch.isinf(top) & (top < 0), torch.zeros_like(top), top)
    w = torch.where(seen, torch.exp(score - base), torch.zeros_like(score))
    total = w.sum(dim=1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink - base)
    return torch.where((total == 0) & ~seen.any(dim=1, keepdim=True), torch.zeros_like(w), w / total), seen


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, first: torch.Tensor, last: torch.Tensor,
           sink: float | None, scale: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Attention of ``weights``' rows over ``v [N, D]``: the sums ``[R, D]``, the sums of ``w |v|`` and the rows' largest
    ``sum |q k| * scale``."""
    w, seen = weights(q, k, first, last, sink, scale)
    finite = torch.isfinite(v)
    out = w @ torch.where(finite, v, torch.zeros_like(v))
    size = w @ torch.where(finite, v.abs(), torch.zeros_like(v))
    for row, dim in (~finite).nonzero().tolist():  # few: added where they are seen
        out[:, dim] += torch.where(seen[:, row], v[row, dim], torch.zeros_like(out[:, dim]))
    reach = torch.where(seen, q.abs() @ k.abs().T.contiguous() * scale, torch.zeros_like(w)).amax(dim=1) if w.shape[1] else w.sum(dim=1)
    return out, size, reach


def prompt_attention(q, k, v, starts, sinks=None, window=None, scale=None):
    """``q [T, H, D]``, ``k``, ``v [T, KV, D]`` of any type, ``starts`` a list -> float64 ``(out, size, reach)`` with
    NaN in rows outside every sequence (``reach [T, H]``)."""
    heads, dim = q.shape[1:]
    group = heads // k.shape[1]
    scale = scale if scale is not None else 1.0 / math.sqrt(dim)
    out = torch.full(q.shape, math.nan, dtype=torch.float64, device=q.device)
    size, reach = out.clone(), out[..., 0].clone()
    for a, b in zip(starts, starts[1:]):
        last = torch.arange(b - a, device=q.device)
        first = (last - window + 1).clamp(min=0) if window else torch.zeros_like(last)
        for h in range(heads):
            if b > a:
                out[a:b, h], size[a:b, h], reach[a:b, h] = attend(
                    q[a:b, h].double(), k[a:b, h // group].double(), v[a:b, h // group].double(), first, last,
                    None if sinks is None else float(sinks[h]), scale)
    return out, size, reach


def largest_weights(q, k, starts, sinks=None, window=None, scale=None):
    """The largest weight of a key in every row of ``prompt_attention``, float64 ``[T, H]`` (NaN outside every sequence)."""
    heads, dim = q.shape[1:]
    group = heads // k.shape[1]
    out = torch.full(q.shape[:2], math.nan, dtype=torch.float64, device=q.device)
    for a, b in zip(starts, starts[1:]):
        last = torch.arange(b - a, device=q.device)
        first = (last - window + 1).clamp(min=0) if window else torch.zeros_like(last)
        for h in range(heads):
            if b > a:
                w, _ = weights(q[a:b, h].double(), k[a:b, h // group].double(), first, last,
                               None if sinks is None else float(sinks[h]), scale if scale is not None else 1.0 / math.sqrt(dim))
                out[a:b, h] = w.amax(dim=1)
    return out


def batch_attention(q, k_pages, v_pages, tables, lengths, prefix_table=None, prefix_len=0, sinks=None, window=None,
                    scale=None):
    """``q [B, H, D]``, pools ``[P, page, KV, D]``, ``tables``, ``lengths`` and ``prefix_table`` lists of numbers ->
    float64 ``(out, size, reach)``."""
    count, heads, dim = q.shape
    page, kv = k_pages.shape[1:3]
    scale = scale if scale is not None else 1.0 / math.sqrt(dim)
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    size, reach = out.clone(), out[..., 0].clone()
    slots = [prefix_table[i // page] * page + i % page for i in range(prefix_len)]
    for b in range(count):
        n = lengths[b]
        if n < 0:
            continue
        at = torch.tensor(slots + [tables[b][i // page] * page + i % page for i in range(n)], dtype=torch.long, device=q.device)
        last = torch.tensor([len(at) - 1], device=q.device)
        first = (last - window + 1).clamp(min=0) if window else torch.zeros_like(last)
        k, v = (x.reshape(-1, kv, dim)[at].double() for x in (k_pages, v_pages))
        for h in range(heads):
            o, s, r = attend(q[b, h:h + 1].double(), k[:, h * kv // heads], v[:, h * kv // heads], first, last,
                             None if sinks is None else float(sinks[h]), scale)
            out[b, h], size[b, h], reach[b, h] = o[0], s[0], r[0]
    return out, size, reach


def tolerance(out, size, reach, keys, dim, p_type, out_type, v_most, top=None):
    """How far float32 work on these sums may be off.  A probability rounded to its type is off by a share of at most
    eps / 2 (and, in float16, by 2^-25 of the row's largest one at least), which moves the sum by that share of
    sum w |v| and, through the normaliser, of |out|; scores summed in float32 are off by at most (dim + 4) 2^-24 of
    sum |q k| scale and move every probability by that, twice; the exponent, its function, the sums over the keys, the
    joins and the division add a share of (keys + 64) 2^-24; the result is rounded by eps / 2 of its type.

    With ``top``, the rows' largest weights of a key, the bound holds relative to small results too.  A float16
    probability is taken relative to a maximum that is at most the largest score, so what it loses below the normal
    range is 2^-25 of ``top`` at most, in the sum and in the normaliser; a result below it loses 2^-25 in float16."""
    u = torch.finfo(p_type).eps / 2
    share = u + 2 * (dim + 4) * 2.0 ** -24 * reach[..., None] * math.exp(1) + (keys + 64) * 2.0 ** -24
    flush = keys * 2.0 ** -25 * v_most if p_type == torch.float16 else 0.0
    if top is not None and p_type == torch.float16:
        flush = keys * 2.0 ** -25 * top[..., None] * (v_most + out.abs())
    near = share * (size + out.abs()) + flush
    if top is not None:
        return near + torch.finfo(out_type).eps / 2 * (out.abs() + near + torch.finfo(out_type).tiny)
    return near + torch.finfo(out_type).eps / 2 * (out.abs() + near) + torch.finfo(out_type).tiny
