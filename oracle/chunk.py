"""Attention of new tokens over a paged cache, the weights they give its keys, and the eviction of the least, in
float64 (test infrastructure only).  A token at key i sees the keys j <= i, with a window those with j > i - window or
j < first."""

from __future__ import annotations

import math

import numpy as np
import torch


def sees(rows: torch.Tensor, keys: torch.Tensor, window: int | None, first: int) -> torch.Tensor:
    """Which of ``keys [N]`` the tokens at ``rows [R]`` see."""
    out = keys[None, :] <= rows[:, None]
    if window:
        out &= (keys[None, :] > rows[:, None] - window) | (keys[None, :] < first)
    return out


def gather(pages: torch.Tensor, table: list[int], n: int) -> torch.Tensor:
    """The first n rows ``[n, KV, D]`` of a sequence's pages, float64."""
    page = pages.shape[1]
    at = torch.tensor([table[i // page] * page + i % page for i in range(n)], dtype=torch.long, device=pages.device)
    return pages.reshape(-1, *pages.shape[2:])[at].double()


def attend(q, k, v, rows, sinks, window, first, scale):
    """``q [R, H, D]`` of the tokens at ``rows [R]`` over ``k``, ``v [N, KV, D]`` -> float64 ``(out, lse, w [R, H, N], size,
    reach)``: the sums, the logs of the normalisers, the weights, the sums of w |v| and the largest sum |q k| scale.  A
    row without a key is zero and its lse the sink, or -inf; scores that are all -inf give NaN.  Values that a row does
    not see do not enter its sum."""
    heads, dim = q.shape[1:]
    n, kv = k.shape[:2]
    group = heads // kv
    seen = sees(rows, torch.arange(n, device=q.device), window, first)
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    size, lse, reach = out.clone(), out[..., 0].clone(), out[..., 0].clone()
    w = torch.zeros((*q.shape[:2], n), dtype=torch.float64, device=q.device)
    for h in range(heads):
        qh, kh, vh = q[:, h].double(), k[:, h // group].contiguous(), v[:, h // group].contiguous()
        score = torch.where(seen, qh @ kh.T.contiguous() * scale, -math.inf)
        sink = -math.inf if sinks is None else float(sinks[h])
        every = torch.cat((score, torch.full((len(rows), 1), sink, dtype=torch.float64, device=q.device)), dim=1)
        top = every.amax(dim=1, keepdim=True)
        base = torch.where(top == -math.inf, torch.zeros_like(top), top)
        e = torch.exp(every - base)
        total = e.sum(dim=1, keepdim=True)
        lse[:, h] = (base + torch.log(total))[:, 0]
        none = ~seen.any(dim=1, keepdim=True)
        p = torch.where(none, torch.zeros_like(score), e[:, :n] / total)
        w[:, h] = torch.where(seen, p, torch.zeros_like(p)) if n else p
        finite = torch.isfinite(vh)
        out[:, h] = p @ torch.where(finite, vh, torch.zeros_like(vh))
        size[:, h] = p.abs() @ torch.where(finite, vh.abs(), torch.zeros_like(vh))
        for row, d in (~finite).nonzero().tolist():  # few: added where they are seen
            out[:, h, d] += torch.where(seen[:, row], vh[row, d], torch.zeros_like(out[:, h, d]))
        if n:
            kf = torch.where(torch.isfinite(kh), kh.abs(), torch.zeros_like(kh))
            reach[:, h] = torch.where(seen, qh.abs() @ kf.T.contiguous() * scale, torch.zeros_like(score)).amax(dim=1)
    return out, lse, w, size, reach


def kept_places(weights: np.ndarray, n: int, keep: int, recent: int, first: int) -> np.ndarray:
    """The old places ``[keep]`` of the keys of a list that stay, place by place (-1 past a short list)."""
    if n <= keep:
        return np.where(np.arange(keep) < n, np.arange(keep), -1)
    ahead = keep - recent
    value = [math.inf if math.isnan(x) else float(x) for x in weights[:n]]
    middle = sorted(range(first, n - recent), key=lambda i: (-value[i], not math.isnan(weights[i]), i))
    stay = set(range(first)) | set(middle[:ahead - first])
    behind = sorted(i for i in stay if i >= ahead)
    out = [i if i in stay else None for i in range(ahead)]
    moved = iter(behind)
    return np.array([next(moved) if i is None else i for i in out] + list(range(n - recent, n)))
