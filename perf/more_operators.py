"""Operators of long conversations over a paged cache, as measurable cases.

Attention of chunks of new tokens (one token of a sequence or many) over the
pages, with a sliding window beside which some first tokens stay visible; the
weights that such queries give the cached keys, summed up key by key; the
eviction of the keys of least weight; and the append of new tokens whose
queries and keys are normalised head by head before they are rotated.  A case
is a dict of plain values; ``run`` takes one operator through one pass, in
elementary torch operations in 32 bits or, where ``own`` is set, through the
framework's entry points.
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
CHUNK = 1 << 28                        # most scores that the plain forms hold at once
EPS = 1e-6


def _chunk(name, sequences, past, new, dtype="fp16", heads=HEADS, kv_heads=KV_HEADS, dim=HEAD_DIM, window=0, first=0,
           sinks=True, page=64, steps=0, past_steps=0, lse=False):
    """`sequences` of up to `past` cached and `new` new tokens, and `steps` beside them of one token behind up to
    `past_steps`."""
    return {"name": name, "kind": "chunk", "sequences": sequences, "past": past, "new": new, "dtype": dtype,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "window": window, "first": first, "sinks": sinks,
            "page": page, "steps": steps, "past_steps": past_steps, "lse": lse}


def _weights(name, sequences, past, new, **more):
    return dict(_chunk(name, sequences, past, new, **more), kind="weights", lse=True)


def _evict(name, layers, sequences, longest, keep, recent, first=4, dtype="fp16", kv_heads=KV_HEADS, dim=HEAD_DIM, page=64):
    return {"name": name, "kind": "evict", "layers": layers, "sequences": sequences, "longest": longest, "keep": keep,
            "recent": recent, "first": first, "dtype": dtype, "kv_heads": kv_heads, "dim": dim, "page": page}


def _append(name, tokens, sequences, dtype="fp16", heads=HEADS, kv_heads=KV_HEADS, dim=HEAD_DIM, page=64, fused=False):
    return {"name": name, "kind": "append", "tokens": tokens, "sequences": sequences, "dtype": dtype, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "fused": fused}


def listed() -> list[dict]:
    return [
        # one decode step of a few conversations whose weights are kept: the call's latency
        _chunk("steps_8", 8, 700, 1, lse=True),
        # questions of a hundred tokens in twelve conversations
        _chunk("suffixes_12x100", 12, 4000, 100),
        # a long prompt's next part beside the steps of 64 other conversations
        _chunk("mixed_6000_64", 1, 2000, 6000, dtype="bf16", steps=64, past_steps=1000),
        # the next part of a long document, larger heads, no sinks
        _chunk("document_d128", 1, 16000, 2000, dtype="bf16", heads=32, kv_heads=8, dim=128, sinks=False, page=16),
        # one step of many endless conversations: the last keys and a few first ones
        _chunk("steps_200_window_first", 200, 2500, 1, window=1024, first=4),
        # the weights of one decode step's keys
        _weights("weights_steps_64", 64, 2000, 1),
        # of a prompt's next part
        _weights("weights_1000", 1, 4000, 1000, dtype="bf16"),
        # a page's worth of keys leaves each of eight full caches, one layer
        _evict("evict_page", 1, 8, 2064, 2000, 128),
        # caches of three conversations cut to a quarter in every layer of the larger model
        _evict("evict_36_layers", 36, 3, 6001, 1500, 256, dtype="bf16"),
        # one decode step's tokens of a batch
        _append("norm_append_64", 64, 64),
        # a prefill step's tokens, q, k and v from one projection, larger heads
        _append("norm_append_6001", 6001, 12, dtype="bf16", heads=32, kv_heads=8, dim=128, fused=True),
    ]


def _log(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    kind = rng.choice(("chunk", "chunk", "chunk", "weights", "weights", "evict", "evict", "append"))
    dtype = rng.choice(("bf16", "fp16"))
    heads, kv_heads, dim = rng.choice(((64, 8, 64), (64, 8, 64), (32, 8, 128), (16, 16, 64), (24, 4, 96), (8, 1, 128),
                                       (28, 4, 80), (20, 5, 48)))
    page = rng.choice((16, 32, 64, 64, 128))
    if kind == "append":
        tokens = _log(rng, 1, 8000)
        case = _append("", tokens, min(tokens, _log(rng, 1, 64)), dtype, heads, kv_heads, dim, page, rng.random() < 0.5)
    elif kind == "evict":
        longest = _log(rng, 40, 12000)
        keep = max(8, round(longest * rng.uniform(0.2, 1.0)))
        recent = min(_log(rng, 1, 512), keep // 2)
        layers = min(rng.choice((1, 1, 2, 12, 36)), max(1, 80000000 // (longest * kv_heads * dim)))
        sequences = _log(rng, 1, max(1, min(64, 80000000 // (layers * longest * kv_heads * dim))))
        case = _evict("", layers, sequences, longest, keep, recent, rng.choice((0, 1, 4, min(32, keep // 4))), dtype,
                      kv_heads, dim, page)
    else:
        window = rng.choice((0, 0, 0, WINDOW, _log(rng, 16, 4096)))
        first = rng.choice((0, 1, 4, _log(rng, 1, 200))) if window else 0
        new = rng.choice((1, _log(rng, 1, 30), _log(rng, 30, 4000)))
        most = max(1, min(200, 4000 // new))
        sequences = _log(rng, 1, most)
        past = rng.choice((0, _log(rng, 16, min(24000, 120000000 // (kv_heads * dim * sequences)))))
        if kind == "chunk":
            steps = rng.choice((0, 0, _log(rng, 1, 64)))
            case = _chunk("", sequences, past, new, dtype, heads, kv_heads, dim, window, first, rng.random() < 0.6, page,
                          steps, _log(rng, 16, 2000) if steps else 0, rng.random() < 0.3)
        else:
            case = _weights("", sequences, past, new, dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim,
                            window=window, first=first, sinks=rng.random() < 0.6, page=page)
    del case["name"]
    return case


# ---- inputs ---------------------------------------------------------------------------


def _int32(values) -> torch.Tensor:
    return torch.tensor(np.ascontiguousarray(values), dtype=torch.int32).cuda()


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape, dtype=torch.bfloat16, std=1.0) -> torch.Tensor:
    return torch.randn(shape, device="cuda", generator=g).mul_(std).to(dtype)


def _chunk_sizes(case) -> tuple[list[int], list[int]]:
    """New tokens and keys, the new ones' among them, of each sequence: uneven, the first the longest."""
    rng = random.Random(1000003 * case["past"] + 1009 * case["new"] + case["sequences"])
    counts, keys = [], []
    for i in range(case["sequences"]):
        n = case["new"] if i == 0 else rng.randint(max(1, case["new"] // 2), case["new"])
        counts.append(n)
        keys.append(n + (case["past"] if i == 0 else rng.randint(case["past"] // 2, case["past"])))
    for _ in range(case["steps"]):
        counts.append(1)
        keys.append(1 + rng.randint(case["past_steps"] // 4, case["past_steps"]))
    order = list(range(len(counts)))
    rng.shuffle(order)
    return [counts[i] for i in order], [keys[i] for i in order]


def _evict_lengths(case) -> list[int]:
    rng = random.Random(1009 * case["longest"] + case["sequences"])
    return [case["longest"]] + [rng.randint((case["longest"] + case["keep"]) // 2, case["longest"])
                                for _ in range(case["sequences"] - 1)]


def _tables(keys, page: int, seed: int) -> tuple[torch.Tensor, int]:
    """Pages of the sequences' keys, in no order, -1 behind them, and the pool's size."""
    held = [-(-n // page) for n in keys]
    n_pages = sum(held) + 3
    order = np.random.RandomState(int(seed) % (1 << 32)).permutation(n_pages)
    tables = np.full((len(keys), max(held)), -1, np.int32)
    at = 0
    for b, n in enumerate(held):
        tables[b, :n] = order[at:at + n]
        at += n
    return _int32(tables), n_pages


def prepare(case, seed):
    g = _gen(seed)
    state = dict(case)
    kv_heads, dim, page = case["kv_heads"], case["dim"], case["page"]
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "evict":
        lengths, layers = _evict_lengths(case), case["layers"]
        tables, n_pages = _tables(lengths, page, seed)
        count, capacity = len(lengths), -(-case["longest"] // page) * page
        # sums of weights: few large ones, many near zero, some never seen, some layers' of one step (many alike)
        weights = torch.randn((layers, count + 2, kv_heads, capacity), device="cuda", generator=g).mul_(2.0).exp_()
        weights.masked_fill_(torch.rand(weights.shape, device="cuda", generator=g) < 0.2, 0.0)
        weights[:, :, kv_heads // 2].mul_(4.0).floor_()
        rows = torch.randperm(count + 2, device="cuda", generator=g)[:count].to(torch.int32)
        pools = torch.empty((2 * layers, n_pages, page, kv_heads, dim), dtype=dtype, device="cuda")
        for pool in pools:
            pool.copy_(torch.randn(pool.shape, device="cuda", generator=g))
        state.update(pools=pools, weights=weights, rows=rows, tables=tables, lengths=_int32(lengths), sizes=lengths)
        return state
    heads = case["heads"]
    if case["kind"] == "append":
        rng = random.Random(1000 * case["tokens"] + case["sequences"])
        tokens, count = case["tokens"], case["sequences"]
        share = [rng.uniform(0.05, 1.0) for _ in range(count)]
        at = [round((tokens - count) * x) for x in np.cumsum([0.0] + share) / sum(share)]
        lengths = [1 + b - a for a, b in zip(at, at[1:])]
        past = [(37 * i) % 1500 for i in range(count)]
        tables, n_pages = _tables([a + n for a, n in zip(past, lengths)], page, seed)
        host = tables.cpu().numpy()
        positions = np.concatenate([np.arange(a, a + n) for a, n in zip(past, lengths)])
        slots = np.concatenate([host[b, np.arange(a, a + n) // page].astype(np.int64) * page + np.arange(a, a + n) % page
                                for b, (a, n) in enumerate(zip(past, lengths))])
        angle = torch.arange(int(positions.max()) + 1, device="cuda").double()[:, None] * (
            150000.0 ** (-torch.arange(dim // 2, device="cuda").double() / (dim // 2)))
        if case["fused"]:
            qkv = _normal(g, tokens, heads + 2 * kv_heads, dim, std=3.0)
            state["q"], state["k"], state["v"] = qkv.split((heads, kv_heads, kv_heads), dim=1)
        else:
            state.update(q=_normal(g, tokens, heads, dim, std=3.0), k=_normal(g, tokens, kv_heads, dim, std=3.0),
                         v=_normal(g, tokens, kv_heads, dim))
        state.update(q_norm=(1.0 + 0.3 * torch.randn(dim, device="cuda", generator=g)).to(torch.bfloat16),
                     k_norm=(1.0 + 0.3 * torch.randn(dim, device="cuda", generator=g)).to(torch.bfloat16),
                     cos=angle.cos().to(torch.bfloat16), sin=angle.sin().to(torch.bfloat16), positions=_int32(positions),
                     slots=_int32(slots), k_pages=_normal(g, n_pages, page, kv_heads, dim, dtype=dtype),
                     v_pages=_normal(g, n_pages, page, kv_heads, dim, dtype=dtype))
        return state
    counts, keys = _chunk_sizes(case)
    tables, n_pages = _tables(keys, page, seed)
    state.update(q=_normal(g, sum(counts), heads, dim, std=2.0), counts=counts, keys=keys, tables=tables,
                 lengths=_int32(keys), k_pages=_normal(g, n_pages, page, kv_heads, dim, dtype=dtype))
    state["sink"] = _normal(g, heads) if case["sinks"] else None
    if case["kind"] == "chunk":
        state["v_pages"] = _normal(g, n_pages, page, kv_heads, dim, dtype=dtype)
    else:
        state["normaliser"] = _plain_chunk(state, values=False)
        capacity = tables.shape[1] * page
        state["weights"] = torch.rand((len(counts) + 1, kv_heads, capacity), device="cuda", generator=g)
        state["rows"] = torch.randperm(len(counts) + 1, device="cuda", generator=g)[:len(counts)].to(torch.int32)
    if own:  # which rows and keys each part of the machine takes: made once a batch, for all layers
        state["plan"] = _ops().attention_plan(counts, keys, heads, kv_heads, dim, window=case["window"] or None,
                                              first=case["first"])
    return state


# ---- one pass -------------------------------------------------------------------------


def _hidden(rows, columns, window: int, first: int):
    """Where a query at position `rows` does not see key `columns`."""
    out = columns > rows
    if window:
        out = out | ((columns <= rows - window) & (columns >= first))
    return out


def _score_blocks(s):
    """Per sequence and block of its new tokens: sequence, first token, tokens, scores [heads, tokens, keys], -inf where
    a token does not see a key."""
    heads, kv_heads, dim = s["heads"], s["kv_heads"], s["dim"]
    group = heads // kv_heads
    start = 0
    # sequences have nothing to do with each other, and the scores of a long one do not fit at once
    for b, (count, n) in enumerate(zip(s["counts"], s["keys"])):
        pages = s["tables"][b, :-(-n // s["page"])].long()
        k = s["k_pages"][pages].float().reshape(-1, kv_heads, dim)[:n].permute(1, 2, 0)
        k = k.repeat_interleave(group, dim=0)
        rows = max(1, min(count, CHUNK // (heads * n)))
        columns = torch.arange(n, device="cuda")[None, :]
        for r0 in range(0, count, rows):
            r1 = min(count, r0 + rows)
            q = s["q"][start + r0:start + r1].float().transpose(0, 1).contiguous()
            scores = torch.bmm(q, k) * (1.0 / math.sqrt(dim))
            position = torch.arange(n - count + r0, n - count + r1, device="cuda")[:, None]
            scores.masked_fill_(_hidden(position, columns, s["window"], s["first"]), -math.inf)
            yield b, start + r0, r1 - r0, pages, n, scores
        start += count


def _steps_scores(s, k):
    """One token of each sequence: scores [sequences, kv heads, group, keys] of padded keys [sequences, keys, kv, dim]."""
    heads, kv_heads, dim = s["heads"], s["kv_heads"], s["dim"]
    count, keys = k.shape[:2]
    q = s["q"].float().reshape(count * kv_heads, heads // kv_heads, dim)
    by_head = k.permute(0, 2, 3, 1).reshape(count * kv_heads, dim, keys).contiguous()
    scores = (torch.bmm(q, by_head) * (1.0 / math.sqrt(dim))).view(count, kv_heads, heads // kv_heads, keys)
    position = s["lengths"].long()[:, None] - 1
    hidden = _hidden(position, torch.arange(keys, device="cuda")[None, :], s["window"], s["first"])
    return scores.masked_fill_(hidden[:, None, None, :], -math.inf)


def _padded(s, pages):
    return pages[s["tables"].long().clamp(min=0)].float().reshape(len(s["counts"]), -1, s["kv_heads"], s["dim"])


def _steps_alone(s) -> bool:
    return max(s["counts"]) == 1 and len(s["counts"]) * s["tables"].shape[1] * s["page"] * s["heads"] <= CHUNK


def _plain_chunk(s, values=True):
    heads, kv_heads, dim = s["heads"], s["kv_heads"], s["dim"]
    group = heads // kv_heads
    sink = None if s["sink"] is None else s["sink"].float()
    lse = torch.empty((s["q"].shape[0], heads), dtype=torch.float32, device="cuda")
    out = torch.empty_like(s["q"]) if values else None

    def softmax_parts(scores, sink):
        m = scores.amax(dim=-1, keepdim=True)
        if sink is not None:
            m = torch.maximum(m, sink)
        p = torch.exp(scores - m)
        total = p.sum(dim=-1, keepdim=True)
        if sink is not None:
            total = total + torch.exp(sink - m)
        return p, total, m + torch.log(total)

    if _steps_alone(s):
        count = len(s["counts"])
        p, total, norm = softmax_parts(_steps_scores(s, _padded(s, s["k_pages"])),
                                       None if sink is None else sink.view(1, kv_heads, group, 1))
        lse.copy_(norm.view(count, heads))
        if values:
            v = _padded(s, s["v_pages"]).transpose(1, 2).reshape(count * kv_heads, -1, dim).contiguous()
            # what no query sees may be anything, NaN included
            seen = torch.arange(v.shape[1], device="cuda")[None, :] < s["lengths"].long()[:, None]
            v = torch.where(seen.repeat_interleave(kv_heads, dim=0)[:, :, None], v, 0.0)
            out.copy_((torch.bmm(p.view(count * kv_heads, group, -1), v).view(count, kv_heads, group, dim) / total)
                      .reshape(count, heads, dim))
    else:
        last, v = -1, None
        for b, row, rows, pages, n, scores in _score_blocks(s):
            p, total, norm = softmax_parts(scores, None if sink is None else sink[:, None, None])
            lse[row:row + rows] = norm[..., 0].T
            if values:
                if b != last:
                    last, v = b, s["v_pages"][pages].float().reshape(-1, kv_heads, dim)[:n].transpose(0, 1)
                    v = v.repeat_interleave(group, dim=0)
                out[row:row + rows] = (torch.bmm(p, v) / total).transpose(0, 1).to(out.dtype)
    if not values:
        return lse
    return (out, lse) if s["lse"] else out


def _plain_weights(s):
    kv_heads, weights, norm = s["kv_heads"], s["weights"], s["normaliser"]
    group = s["heads"] // kv_heads
    at = s["rows"].long()
    if _steps_alone(s):
        count, keys = len(s["counts"]), s["tables"].shape[1] * s["page"]
        p = torch.exp(_steps_scores(s, _padded(s, s["k_pages"])) - norm.view(count, kv_heads, group, 1)).sum(dim=2)
        end = s["lengths"].long()[:, None, None]
        column = torch.arange(keys, device="cuda")
        held = weights[at]
        held = torch.where(column < end - 1, held + p, torch.where(column == end - 1, p, held))
        weights[at] = held
        return weights
    last, held = -1, None
    for b, row, rows, pages, n, scores in _score_blocks(s):
        p = torch.exp(scores - norm[row:row + rows].T[:, :, None])
        p = p.view(kv_heads, group, rows, n).sum(dim=(1, 2), dtype=torch.float64)
        if b != last:
            if last >= 0:
                weights[at[last], :, :held.shape[1]] = held.float()
            last, held = b, weights[at[b], :, :n].double()
            held[:, n - s["counts"][b]:] = 0.0
        held += p
    weights[at[last], :, :held.shape[1]] = held.float()
    return weights


def _kept(weights, n: int, keep: int, recent: int, first: int):
    """Rows of weights [..., >= n] -> the old places [..., keep] of the keys that stay, place by place."""
    ahead, column = keep - recent, torch.arange(n, device=weights.device)
    value = weights[..., :n].clone()
    value[..., :first] = math.inf          # always kept, in front of all others
    value[..., n - recent:] = -math.inf    # placed by themselves
    stays = torch.zeros(value.shape, dtype=torch.bool, device=weights.device)
    order = torch.sort(value[..., :n - recent], dim=-1, descending=True, stable=True).indices[..., :ahead]
    stays.scatter_(-1, order, True)
    holes, moved = ~stays[..., :ahead], stays[..., ahead:]
    out = column[:keep].expand(*value.shape[:-1], keep).clone()
    out[..., ahead:] = column[n - recent:]
    # the i-th hole takes the i-th kept key from behind: as many of the one as of the other in every row
    out[..., :ahead][holes] = column[ahead:].expand(moved.shape)[moved]
    return out


def _plain_evict(s):
    pools, weights, keep, recent, first, page = s["pools"], s["weights"], s["keep"], s["recent"], s["first"], s["page"]
    layers, kv_heads, dim = s["layers"], s["kv_heads"], s["dim"]
    kept = torch.full((layers, len(s["sizes"]), kv_heads, keep), -1, dtype=torch.int32, device="cuda")
    heads = torch.arange(kv_heads, device="cuda")[:, None]
    for b, n in enumerate(s["sizes"]):
        if n <= keep:
            kept[:, b, :, :n] = torch.arange(n, dtype=torch.int32, device="cuda")
            continue
        row, table = s["rows"][b].long(), s["tables"][b].long()
        held = weights[:, row]                                   # [layers, kv, capacity], a copy
        old = _kept(held, n, keep, recent, first)                # [layers, kv, keep]
        kept[:, b] = old
        weights[:, row, :, :keep] = torch.gather(held, -1, old)
        new = torch.arange(keep, device="cuda")[None, :]
        for layer in range(layers):
            for pool in pools[2 * layer:2 * layer + 2]:
                pool[table[new // page], new % page, heads] = pool[table[old[layer] // page], old[layer] % page, heads]
    return kept, weights, pools


def _plain_append(s):
    cos, sin = (s[n][s["positions"].long()].float()[:, None, :] for n in ("cos", "sin"))

    def turned(x, weight):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * weight.float()
        a, b = x.chunk(2, dim=-1)
        return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)

    q, k = turned(s["q"], s["q_norm"]), turned(s["k"], s["k_norm"])
    at = s["slots"].long()
    shape = (-1, s["kv_heads"], s["dim"])
    s["k_pages"].view(shape)[at] = k.to(s["k_pages"].dtype)
    s["v_pages"].view(shape)[at] = s["v"].float().to(s["v_pages"].dtype)
    return q.to(s["q"].dtype), k.to(s["k"].dtype), s["k_pages"], s["v_pages"]


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
        if kind == "chunk":
            return ops.chunk_attention(s["q"], s["k_pages"], s["v_pages"], s["tables"], s["lengths"], s["plan"],
                                       sinks=s["sink"], want_lse=s["lse"])
        if kind == "weights":
            ops.add_key_weights(s["q"], s["normaliser"], s["k_pages"], s["tables"], s["lengths"], s["plan"],
                                s["weights"], s["rows"])
            return s["weights"]
        if kind == "evict":
            kept = ops.evict_keys(s["pools"], s["weights"], s["tables"], s["lengths"], s["rows"], s["keep"],
                                  recent=s["recent"], first=s["first"])
            return kept, s["weights"], s["pools"]
        q, k = ops.paged_append(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["positions"], s["slots"], s["k_pages"],
                                s["v_pages"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
        return q, k, s["k_pages"], s["v_pages"]
    return {"chunk": _plain_chunk, "weights": _plain_weights, "evict": _plain_evict, "append": _plain_append}[kind](s)


# ---- what a pass cannot do without ----------------------------------------------------


def _pairs(count: int, n: int, window: int, first: int) -> int:
    """Pairs of a new token and a key that it sees."""
    p = np.arange(n - count, n, dtype=np.int64)
    if not window:
        return int((p + 1).sum())
    low = np.maximum(p + 1 - window, 0)
    return int((p + 1 - low + np.minimum(low, first)).sum())


def _seen_keys(count: int, n: int, window: int, first: int) -> int:
    low = max(0, n - count + 1 - window) if window else 0
    return n - low + min(low, first)


def work(case):
    kv_heads, dim = case["kv_heads"], case["dim"]
    if case["kind"] == "evict":
        moved = weights = 0.0
        for n in _evict_lengths(case):
            if n > case["keep"]:
                # weights that have nothing to do with their places: a kept key is behind the middle's end as often as any
                middle, stay = n - case["recent"] - case["first"], case["keep"] - case["recent"] - case["first"]
                moved += case["recent"] + max(0, stay) * (n - case["keep"]) / max(1, middle)
                weights += n + 2 * case["keep"]
        lists = case["layers"] * kv_heads
        return {"bytes": int(lists * (moved * 2 * 2 * 2 * dim + 4 * weights)), "flops": 0}
    heads = case["heads"]
    if case["kind"] == "append":
        n = case["tokens"]
        return {"bytes": 2 * n * dim * (2 * heads + 5 * kv_heads) + n * (2 * dim + 8),
                "flops": n * dim * (7 * (heads + kv_heads))}
    sizes = [(c, n, case["window"], case["first"]) for c, n in zip(*_chunk_sizes(case))]
    tokens, keys, pairs = sum(c for c, *_ in sizes), sum(_seen_keys(*x) for x in sizes), sum(_pairs(*x) for x in sizes)
    if case["kind"] == "weights":
        return {"bytes": 2 * kv_heads * dim * keys + 8 * kv_heads * keys + tokens * heads * (2 * dim + 4),
                "flops": 2 * heads * dim * pairs}
    return {"bytes": 4 * kv_heads * dim * keys + tokens * heads * (4 * dim + (4 if case["lse"] else 0)),
            "flops": 4 * heads * dim * pairs}


# ---- the definition in 64 bits --------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    kind, kv_heads, dim, page = case["kind"], case["kv_heads"], case["dim"], case["page"]
    if kind == "evict":
        return _exact_evict(case, s)
    heads = case["heads"]
    group = heads // kv_heads
    if kind == "append":
        half, at = dim // 2, s["positions"].long()
        unit = torch.complex(s["cos"].double()[at], s["sin"].double()[at])[:, None, :]

        def turn(x, weight):
            y = x.double()
            y = y / torch.sqrt(torch.square(y).sum(-1, keepdim=True) / dim + EPS) * weight.double()
            z = torch.complex(y[..., :half].contiguous(), y[..., half:].contiguous()) * unit
            return torch.cat((z.real, z.imag), dim=-1)

        q, k = turn(s["q"], s["q_norm"]), turn(s["k"], s["k_norm"])
        slots = s["slots"].long()
        k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
        k_pages.index_put_((slots // page, slots % page), k)
        v_pages.index_put_((slots // page, slots % page), s["v"].double())
        return q, k, k_pages, v_pages
    counts, lengths = _chunk_sizes(case)
    if sum(c * n for c, n in zip(counts, lengths)) * heads > 1 << 33:
        return None
    window, first = case["window"], case["first"]
    tokens = sum(counts)
    sink = None if s["sink"] is None else s["sink"].double()
    out = torch.zeros((tokens, heads, dim), dtype=torch.float64, device="cuda")
    lse = torch.zeros((tokens, heads), dtype=torch.float64, device="cuda")
    sums = s["weights"].double() if kind == "weights" else None
    start = 0
    for b, (count, n) in enumerate(zip(counts, lengths)):
        table = s["tables"][b, :-(-n // page)].long()
        if kind == "weights":
            sums[int(s["rows"][b]), :, n - count:n] = 0.0
        for h in range(kv_heads):
            k = s["k_pages"][table, :, h].reshape(-1, dim)[:n].double().T.contiguous()
            v = s["v_pages"][table, :, h].reshape(-1, dim)[:n].double() if kind == "chunk" else None
            step = max(1, (1 << 26) // (group * n))
            for r0 in range(0, count, step):
                r1 = min(count, r0 + step)
                rows = slice(start + r0, start + r1)
                q = s["q"][rows, h * group:(h + 1) * group].double()
                e = (q.reshape(-1, dim) @ k).view(r1 - r0, group, n) / math.sqrt(dim)
                i = torch.arange(n - count + r0, n - count + r1, device="cuda")[:, None]
                j = torch.arange(n, device="cuda")[None, :]
                seen = j <= i
                if window:
                    seen = seen & ((j > i - window) | (j < first))
                e = torch.where(seen[:, None, :], e, torch.full((), -math.inf, dtype=torch.float64, device="cuda"))
                if kind == "weights":
                    norm = s["normaliser"][rows, h * group:(h + 1) * group].double()
                    sums[int(s["rows"][b]), h, :n] += torch.exp(e - norm[..., None]).sum(dim=(0, 1))
                    continue
                if sink is not None:
                    e = torch.cat((e, sink[h * group:(h + 1) * group].view(1, group, 1).expand(r1 - r0, group, 1)), dim=-1)
                lse[rows, h * group:(h + 1) * group] = torch.logsumexp(e, dim=-1)
                w = torch.softmax(e, dim=-1)[..., :n].reshape(-1, n)
                out[rows, h * group:(h + 1) * group] = (w @ v).view(r1 - r0, group, dim)
        start += count
    if kind == "weights":
        return sums
    return (out, lse) if case["lse"] else out


def _exact_evict(case, s):
    keep, recent, first, page = case["keep"], case["recent"], case["first"], case["page"]
    layers, kv_heads = case["layers"], case["kv_heads"]
    weights = s["weights"].cpu().numpy()
    tables, rows = s["tables"].cpu().numpy(), s["rows"].cpu().numpy()
    lengths = _evict_lengths(case)
    kept = np.full((layers, len(lengths), kv_heads, keep), -1, np.int32)
    new_weights = weights.astype(np.float64)
    pools = s["pools"].double()
    for b, n in enumerate(lengths):
        if n <= keep:
            kept[:, b, :, :n] = np.arange(n)
            continue
        for layer in range(layers):
            for h in range(kv_heads):
                w = weights[layer, rows[b], h]
                middle = np.arange(first, n - recent)
                best = np.lexsort((middle, -w[first:n - recent]))[:keep - recent - first]
                stay = np.concatenate((np.arange(min(first, keep - recent)), middle[best]))
                place = np.full(keep, -1)
                place[stay[stay < keep - recent]] = stay[stay < keep - recent]
                place[np.flatnonzero(place[:keep - recent] < 0)] = np.sort(stay[stay >= keep - recent])
                place[keep - recent:] = np.arange(n - recent, n)
                kept[layer, b, h] = place
                new_weights[layer, rows[b], h, :keep] = w[place]
                old, new = torch.from_numpy(place).cuda(), torch.arange(keep, device="cuda")
                table = torch.from_numpy(tables[b]).cuda().long()
                for pool in (pools[2 * layer], pools[2 * layer + 1]):
                    pool[table[new // page], new % page, h] = pool[table[old // page], old % page, h]
    return (torch.from_numpy(kept).cuda(), torch.from_numpy(new_weights).cuda(), pools)
