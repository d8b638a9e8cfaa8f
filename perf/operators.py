"""Operators of a server that holds many sequences, as measurable cases.

Prompt attention (whole prompts, packed, causal), the append of rotated keys
and values to a paged cache, attention of a decode batch over such pages with
a prefix that all its sequences share, and the page copies of forks and
compaction.  A case is a dict of plain values; ``run`` takes one operator
through one pass, in elementary torch operations in 32 bits or, where ``own``
is set, through the framework's entry points.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

HEADS, KV_HEADS, HEAD_DIM = 64, 8, 64  # the model shape of this repository's attention benchmark
WINDOW = 128                           # its sliding layers
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
CHUNK = 1 << 28                        # most scores that the plain prompt form holds at once


def _prompt(name, tokens, sequences, dtype="bf16", heads=HEADS, kv_heads=KV_HEADS, dim=HEAD_DIM, window=0, sinks=True,
            fused=False):
    return {"name": name, "kind": "prompt", "tokens": tokens, "sequences": sequences, "dtype": dtype, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "window": window, "sinks": sinks, "fused": fused}


def _batch(name, sequences, prefix, most_own, dtype="fp16", heads=HEADS, kv_heads=KV_HEADS, dim=HEAD_DIM, window=0,
           sinks=True, page=64):
    return {"name": name, "kind": "batch", "sequences": sequences, "prefix": prefix, "most_own": most_own,
            "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim, "window": window, "sinks": sinks,
            "page": page}


def _append(name, tokens, sequences, dtype="fp16", heads=HEADS, kv_heads=KV_HEADS, dim=HEAD_DIM, page=64):
    return {"name": name, "kind": "append", "tokens": tokens, "sequences": sequences, "dtype": dtype, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page}


def _copy(name, layers, pages, moves, dtype="fp16", kv_heads=KV_HEADS, dim=HEAD_DIM, page=64):
    return {"name": name, "kind": "copy", "layers": layers, "pages": pages, "moves": moves, "dtype": dtype,
            "kv_heads": kv_heads, "dim": dim, "page": page}


def listed() -> list[dict]:
    return [
        # one short question: the call's latency
        _prompt("prompt_97", 97, 1),
        # a prefill step of several requests of different lengths, on a sliding layer, q, k and v from one projection
        _prompt("prompt_packed_window", 6001, 12, window=WINDOW, fused=True),
        # one long document on a full layer
        _prompt("prompt_8192", 8192, 1),
        # two prompts of a model with larger heads, no sinks
        _prompt("prompt_d128", 6778, 2, dtype="fp16", heads=32, kv_heads=8, dim=128, sinks=False),
        # a few answers of one short system prompt: latency
        _batch("batch_8_prefix_500", 8, 500, 40, dtype="bf16"),
        # many users of one long system prompt, each some turns in
        _batch("batch_64_prefix_8192", 64, 8192, 700),
        # the same on a sliding layer, with longer conversations
        _batch("batch_200_window", 200, 1000, 2000, window=WINDOW),
        # questions about one long document, larger heads
        _batch("batch_32_d128", 32, 16000, 900, dtype="bf16", heads=32, kv_heads=8, dim=128, sinks=False, page=16),
        # one decode step's tokens of a batch
        _append("append_64", 64, 64),
        # a prefill step's tokens
        _append("append_6001", 6001, 12, dtype="bf16"),
        # sixteen sequences forked in the middle of a page, in every layer of the larger model
        _copy("fork_16", 36, 64, 16),
        # a compaction of four layers' pages
        _copy("compact_400", 4, 1024, 400, dtype="bf16"),
    ]


def _log(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    kind = rng.choice(("prompt", "prompt", "prompt", "batch", "batch", "batch", "append", "copy"))
    dtype = rng.choice(("bf16", "fp16"))
    heads, kv_heads, dim = rng.choice(((64, 8, 64), (64, 8, 64), (32, 8, 128), (16, 16, 64), (24, 4, 96), (8, 1, 128),
                                       (28, 4, 80), (20, 5, 48)))
    sinks = rng.random() < 0.6
    page = rng.choice((16, 32, 64, 64, 128))
    if kind == "prompt":
        window = rng.choice((0, 0, WINDOW, _log(rng, 16, 4096)))
        tokens = _log(rng, 1, 8000)
        case = _prompt("", tokens, min(tokens, _log(rng, 1, 24)), dtype, heads, kv_heads, dim, window, sinks,
                       rng.random() < 0.5)
    elif kind == "batch":
        window = rng.choice((0, 0, WINDOW, _log(rng, 16, 4096)))
        sequences = _log(rng, 1, 200)
        case = _batch("", sequences, rng.choice((0, _log(rng, 16, 16000))), _log(rng, 1, 100000 // max(50, sequences)),
                      dtype, heads, kv_heads, dim, window, sinks, page)
    elif kind == "append":
        tokens = _log(rng, 1, 8000)
        case = _append("", tokens, min(tokens, _log(rng, 1, 64)), dtype, heads, kv_heads, dim, page)
    else:
        row = kv_heads * dim * page
        pages = min(_log(rng, 8, 4096), (1 << 27) // row)
        layers = rng.randint(1, max(1, min(36, (1 << 27) // (pages * row))))
        most = min(0.45, 50e6 / (layers * pages * row))
        case = _copy("", layers, pages, max(1, round(pages * rng.uniform(0.02, most))), dtype, kv_heads, dim, page)
    del case["name"]
    return case


# ---- inputs ---------------------------------------------------------------------------


def _lengths(case) -> list[int]:
    """The sequences' lengths, at least one token each, uneven, in no order."""
    n, total = case["sequences"], case["tokens"]
    rng = random.Random(1000 * total + n)
    share = [rng.uniform(0.05, 1.0) for _ in range(n)]
    at = [round((total - n) * x) for x in np.cumsum([0.0] + share) / sum(share)]
    return [1 + b - a for a, b in zip(at, at[1:])]


def _own_lengths(case) -> list[int]:
    rng = random.Random(1000 * case["most_own"] + case["sequences"])
    most = case["most_own"]
    return [most] + [rng.randint(max(1, most // 8), most) for _ in range(case["sequences"] - 1)]


def _int32(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32).cuda()


def _normal(g, *shape, dtype=torch.bfloat16, std=1.0) -> torch.Tensor:
    return torch.randn(shape, device="cuda", generator=g).mul_(std).to(dtype)


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(int(seed))


def prepare(case, seed):
    g = _gen(seed)
    state = dict(case)
    if case["kind"] == "copy":
        shape = (2 * case["layers"], case["pages"], case["page"], case["kv_heads"], case["dim"])
        order = np.random.RandomState(int(seed) % (1 << 32)).permutation(case["pages"])
        n = min(case["moves"], case["pages"] // 2)
        state.update(pool=_normal(g, *shape, dtype=DTYPES[case["dtype"]]), src=order[:n].astype(np.int32),
                     dst=order[n:2 * n].astype(np.int32))
        return state
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "batch":
        lengths, page = _own_lengths(case), case["page"]
        width = -(-max(lengths) // page)
        held = [-(-n // page) for n in lengths]
        prefix_pages = -(-case["prefix"] // page)
        n_pages = sum(held) + prefix_pages + 3
        order = torch.randperm(n_pages, device="cuda", generator=g).to(torch.int32)
        tables = torch.zeros((case["sequences"], width), dtype=torch.int32, device="cuda")
        for b, at in enumerate(np.cumsum([prefix_pages] + held[:-1]).tolist()):
            tables[b, :held[b]] = order[at:at + held[b]]
        state.update(q=_normal(g, case["sequences"], heads, dim, std=2.0),
                     k_pages=_normal(g, n_pages, page, kv_heads, dim, dtype=dtype),
                     v_pages=_normal(g, n_pages, page, kv_heads, dim, dtype=dtype), tables=tables,
                     lengths=_int32(lengths), prefix_table=order[:prefix_pages].contiguous())
        state["sink"] = _normal(g, heads) if case["sinks"] else None
        return state
    lengths = _lengths(case)
    tokens = case["tokens"]
    starts = np.cumsum([0] + lengths)
    if case["kind"] == "prompt":
        if case["fused"]:
            qkv = _normal(g, tokens, heads + 2 * kv_heads, dim, dtype=dtype)
            state["q"], state["k"], state["v"] = qkv.split((heads, kv_heads, kv_heads), dim=1)
        else:
            state.update(q=_normal(g, tokens, heads, dim, dtype=dtype), k=_normal(g, tokens, kv_heads, dim, dtype=dtype),
                         v=_normal(g, tokens, kv_heads, dim, dtype=dtype))
        state.update(lengths=lengths, starts=_int32(starts), sink=_normal(g, heads) if case["sinks"] else None)
        return state
    # append: the tokens continue sequences that hold some tokens already
    page = case["page"]
    past = [(37 * i) % 1500 for i in range(len(lengths))]
    held = [-(-(a + n) // page) for a, n in zip(past, lengths)]
    n_pages = sum(held) + 2
    order = np.random.RandomState(int(seed) % (1 << 32)).permutation(n_pages)
    first = np.cumsum([0] + held)
    positions = np.concatenate([np.arange(a, a + n) for a, n in zip(past, lengths)])
    slots = np.concatenate([order[f + np.arange(a, a + n) // page] * page + np.arange(a, a + n) % page
                            for f, a, n in zip(first, past, lengths)])
    angle = torch.arange(max(a + n for a, n in zip(past, lengths)), device="cuda").double()[:, None] * (
        150000.0 ** (-torch.arange(dim // 2, device="cuda").double() / (dim // 2)))
    state.update(q=_normal(g, tokens, heads, dim), k=_normal(g, tokens, kv_heads, dim), v=_normal(g, tokens, kv_heads, dim),
                 cos=angle.cos().to(torch.bfloat16), sin=angle.sin().to(torch.bfloat16), positions=_int32(positions),
                 slots=_int32(slots), k_pages=_normal(g, n_pages, page, kv_heads, dim, dtype=dtype),
                 v_pages=_normal(g, n_pages, page, kv_heads, dim, dtype=dtype))
    return state


# ---- one pass -------------------------------------------------------------------------


def _softmax_sum(scores, values, sink):
    """Rows of scores [heads, rows, keys], -inf where masked, and values [heads, keys, dim] -> their sums."""
    m = scores.amax(dim=-1, keepdim=True)
    if sink is not None:
        m = torch.maximum(m, sink[:, None, None])
    p = torch.exp(scores - m)
    total = p.sum(dim=-1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink[:, None, None] - m)
    return torch.bmm(p, values) / total


def _plain_prompt(s):
    heads, kv_heads, dim, window = s["heads"], s["kv_heads"], s["dim"], s["window"]
    group = heads // kv_heads
    out = torch.empty((s["tokens"], heads, dim), dtype=s["q"].dtype, device="cuda")
    sink = None if s["sink"] is None else s["sink"].float()
    start = 0
    # sequences have nothing to do with each other, and the scores of a long one do not fit at once
    for n in s["lengths"]:
        rows = max(1, min(n, CHUNK // (heads * n)))
        for r0 in range(0, n, rows):
            r1 = min(n, r0 + rows)
            j0 = max(0, r0 - window + 1) if window else 0
            q = s["q"][start + r0:start + r1].float().transpose(0, 1).contiguous()
            k = s["k"][start + j0:start + r1].float().permute(1, 2, 0).repeat_interleave(group, dim=0)
            v = s["v"][start + j0:start + r1].float().transpose(0, 1).repeat_interleave(group, dim=0)
            scores = torch.bmm(q, k) * (1.0 / math.sqrt(dim))
            i = torch.arange(r0, r1, device="cuda")[:, None]
            j = torch.arange(j0, r1, device="cuda")[None, :]
            hidden = (j > i) | (j <= i - window) if window else j > i
            scores.masked_fill_(hidden, -math.inf)
            out[start + r0:start + r1] = _softmax_sum(scores, v, sink).transpose(0, 1).to(out.dtype)
        start += n
    return out


def _plain_batch(s):
    heads, kv_heads, dim, window, prefix = s["heads"], s["kv_heads"], s["dim"], s["window"], s["prefix"]
    group, count, page = heads // kv_heads, s["sequences"], s["page"]
    table = s["tables"].long()
    own_keys = table.shape[1] * page

    def rows(pages, to):
        shared = pages[s["prefix_table"].long()].float().reshape(-1, kv_heads, dim)[:prefix]
        mine = pages[table].float().reshape(count, own_keys, kv_heads, dim)
        if to == "scores":  # [kv, dim, prefix], [count * kv, dim, own]
            return (shared.permute(1, 2, 0).contiguous(),
                    mine.permute(0, 2, 3, 1).reshape(count * kv_heads, dim, own_keys).contiguous())
        return (shared.transpose(0, 1).contiguous(),
                mine.transpose(1, 2).reshape(count * kv_heads, own_keys, dim).contiguous())

    q = s["q"].float().view(count, kv_heads, group, dim)
    by_head = q.transpose(0, 1).reshape(kv_heads, count * group, dim)
    k_shared, k_own = rows(s["k_pages"], "scores")
    c = 1.0 / math.sqrt(dim)
    a = torch.bmm(by_head, k_shared).view(kv_heads, count, group, prefix).transpose(0, 1) * c
    b = torch.bmm(q.reshape(count * kv_heads, group, dim), k_own).view(count, kv_heads, group, own_keys) * c
    scores = torch.cat((a, b), dim=-1)
    j = torch.arange(prefix + own_keys, device="cuda")[None, :]
    end = prefix + s["lengths"].long()[:, None]
    hidden = (j >= end) | (j < end - window) if window else j >= end
    scores = scores.masked_fill(hidden[:, None, None, :], -math.inf)
    m = scores.amax(dim=-1, keepdim=True)
    sink = None
    if s["sink"] is not None:
        sink = s["sink"].float().view(1, kv_heads, group, 1)
        m = torch.maximum(m, sink)
    p = torch.exp(scores - m)
    total = p.sum(dim=-1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink - m)
    v_shared, v_own = rows(s["v_pages"], "sums")
    pa = p[..., :prefix].transpose(0, 1).reshape(kv_heads, count * group, prefix)
    pb = p[..., prefix:].reshape(count * kv_heads, group, own_keys)
    out = (torch.bmm(pa, v_shared).view(kv_heads, count, group, dim).transpose(0, 1)
           + torch.bmm(pb, v_own).view(count, kv_heads, group, dim)) / total
    return out.reshape(count, heads, dim).to(s["q"].dtype)


def _plain_append(s):
    cos, sin = (s[n][s["positions"].long()].float()[:, None, :] for n in ("cos", "sin"))

    def turned(x):
        a, b = x.float().chunk(2, dim=-1)
        return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)

    q, k = turned(s["q"]), turned(s["k"])
    at = s["slots"].long()
    shape = (-1, s["kv_heads"], s["dim"])
    s["k_pages"].view(shape)[at] = k.to(s["k_pages"].dtype)
    s["v_pages"].view(shape)[at] = s["v"].float().to(s["v_pages"].dtype)
    return q.to(s["q"].dtype), k.to(s["k"].dtype), s["k_pages"], s["v_pages"]


def _plain_copy(s):
    src, dst = (torch.from_numpy(s[n]).cuda().long() for n in ("src", "dst"))
    s["pool"][:, dst] = s["pool"][:, src]
    return s["pool"]


_entry_points = None


def _ops():
    global _entry_points
    if _entry_points is None:
        root = str(Path(__file__).resolve().parents[1] / "kcapw-klcquant_amd")
        if root not in sys.path:
            sys.path.insert(0, root)
        from klcquant_amd import ops as _entry_points
    return _entry_points


def run(s):
    kind = s["kind"]
    if own:
        ops = _ops()
        if kind == "prompt":
            return ops.prompt_attention(s["q"], s["k"], s["v"], s["starts"], sinks=s["sink"], window=s["window"] or None)
        if kind == "batch":
            return ops.batch_attention(s["q"], s["k_pages"], s["v_pages"], s["tables"], s["lengths"],
                                       prefix_table=s["prefix_table"], prefix_len=s["prefix"], sinks=s["sink"],
                                       window=s["window"] or None)
        if kind == "append":
            q, k = ops.paged_append(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["positions"], s["slots"], s["k_pages"],
                                    s["v_pages"])
            return q, k, s["k_pages"], s["v_pages"]
        ops.copy_pages(s["pool"], s["src"], s["dst"])
        return s["pool"]
    return {"prompt": _plain_prompt, "batch": _plain_batch, "append": _plain_append, "copy": _plain_copy}[kind](s)


# ---- what a pass cannot do without ----------------------------------------------------


def _visible(n: int, window: int) -> int:
    """Pairs of a query and a visible key in a causal sequence of n tokens."""
    if not window or window >= n:
        return n * (n + 1) // 2
    return window * (window + 1) // 2 + (n - window) * window


def work(case):
    if case["kind"] == "copy":
        row = 2 * case["page"] * case["kv_heads"] * case["dim"]
        return {"bytes": 2 * 2 * case["layers"] * min(case["moves"], case["pages"] // 2) * row, "flops": 0}
    heads, kv_heads, dim, w = case["heads"], case["kv_heads"], case["dim"], case.get("window", 0)
    if case["kind"] == "append":
        n = case["tokens"]
        return {"bytes": 2 * n * dim * (2 * heads + 5 * kv_heads) + n * (2 * dim + 8),
                "flops": 3 * n * dim * (heads + kv_heads)}
    if case["kind"] == "prompt":
        n = case["tokens"]
        return {"bytes": 2 * n * dim * (2 * heads + 2 * kv_heads),
                "flops": 4 * heads * dim * sum(_visible(x, w) for x in _lengths(case))}
    lengths, prefix = _own_lengths(case), case["prefix"]
    own_keys = [min(n, w) if w else n for n in lengths]
    shared = [min(prefix, max(0, w - n)) if w else prefix for n in lengths]
    return {"bytes": 2 * (2 * kv_heads * dim * (sum(own_keys) + max(shared)) + 2 * len(lengths) * heads * dim),
            "flops": 4 * heads * dim * (sum(own_keys) + sum(shared))}


# ---- the definition in 64 bits --------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "copy":
        out = s["pool"].double()
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            out[:, b].copy_(out[:, a])
        return out
    if kind == "append":
        half = case["dim"] // 2
        at = s["positions"].long()
        unit = torch.complex(s["cos"].double()[at], s["sin"].double()[at])[:, None, :]

        def turn(x):
            z = torch.complex(x[..., :half].double(), x[..., half:].double()) * unit
            return torch.cat((z.real, z.imag), dim=-1)

        q, k = turn(s["q"]), turn(s["k"])
        page = case["page"]
        slots = s["slots"].long()
        k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
        k_pages.index_put_((slots // page, slots % page), k)
        v_pages.index_put_((slots // page, slots % page), s["v"].double())
        return q, k, k_pages, v_pages
    heads, kv_heads, dim, window = case["heads"], case["kv_heads"], case["dim"], case["window"]
    group = heads // kv_heads
    sink = None if s["sink"] is None else s["sink"].double()

    def attend(q, k, v, positions, first, head):
        """Rows of one head: q [rows, dim] at `positions`, keys and values [keys, dim] from position `first` on."""
        e = (q @ k.T.contiguous()) / math.sqrt(dim)
        j = torch.arange(first, first + k.shape[0], device="cuda")
        seen = j[None, :] <= positions[:, None]
        if window:
            seen &= j[None, :] > positions[:, None] - window
        e = torch.where(seen, e, torch.full_like(e, -math.inf))
        if sink is not None:
            e = torch.cat((e, sink[head].expand(e.shape[0], 1)), dim=1)
        w = torch.softmax(e, dim=1)
        return w[:, :k.shape[0]] @ v

    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    if kind == "prompt":
        start = 0
        for n in _lengths(case):
            for h in range(heads):
                k, v = (s[x][start:start + n, h // group].double() for x in ("k", "v"))
                for r0 in range(0, n, 4096):
                    r1 = min(n, r0 + 4096)
                    first = max(0, r0 - window + 1) if window else 0
                    out[start + r0:start + r1, h] = attend(s["q"][start + r0:start + r1, h].double(), k[first:r1],
                                                           v[first:r1], torch.arange(r0, r1, device="cuda"), first, h)
            start += n
        return out
    prefix, page = case["prefix"], case["page"]
    shared = [s[x][s["prefix_table"].long()].flatten(0, 1)[:prefix].double() for x in ("k_pages", "v_pages")]
    for b, n in enumerate(_own_lengths(case)):
        pages = s["tables"][b, :-(-n // page)].long()
        k, v = (torch.cat((a, s[x][pages].flatten(0, 1)[:n].double())) for a, x in zip(shared, ("k_pages", "v_pages")))
        for kv in range(kv_heads):
            kk, vv = k[:, kv].contiguous(), v[:, kv].contiguous()
            q = s["q"][b, kv * group:(kv + 1) * group].double()
            e = (q @ kk.T.contiguous()) / math.sqrt(dim)
            if window:
                e[:, :max(0, int(prefix + n - window))] = -math.inf
            if sink is not None:
                e = torch.cat((e, sink[kv * group:(kv + 1) * group, None]), dim=1)
            out[b, kv * group:(kv + 1) * group] = torch.softmax(e, dim=1)[:, :kk.shape[0]] @ vv
    return out
