"""A KV cache of many sequences in pages, and the attention layer over it.

``PageTable``         which sequence holds which pages: host bookkeeping alone.
``PagedKVCache``      a PageTable with its pages in HBM, one slab for all
                      layers' keys and values, so that a fork or a compaction
                      is one launch (ops.copy_pages) whatever the number of
                      layers.
``BatchedAttention``  StreamedAttention's layer (projections, RoPE, sinks,
                      window) for a batch of tokens of several sequences:
                      whole prompts by ops.prompt_attention, steps of one
                      token a sequence by ops.batch_attention, where pages
                      that all of them share are read once on layers without
                      a window, if they are many, and suffixes of several
                      tokens, alone or beside steps, by ops.chunk_attention.
                      So are all tokens that see some first ones beside their
                      window, and all of a cache that keeps weights.

A cache may keep the weights that its keys were given, layer by layer and head
by head, and evict the keys of the least (ops.add_key_weights, ops.evict_keys):
sequences of any number of tokens then stay within a number of keys.

Pages are shared while they are full and never written then: a fork takes its
parent's full pages as they are and a copy of the last one, and an eviction
writes to copies.  Work on the cache is ordered by the stream it runs on; a
caller with several streams orders them.
"""

from __future__ import annotations

import operator
from dataclasses import dataclass, field

import numpy as np
import torch

from . import ops
from .attention import _KV_DTYPES, AttentionConfig, yarn_attention_scaling, yarn_inv_freq


_MAX_ROWS = 65535  # of a batch_attention call
_ALL = 1 << 30     # more than a sequence has


class PageTable:
    """Pages of ``page_size`` tokens among sequences, numbered as they were added (numbers are used again)."""

    def __init__(self, n_pages: int, page_size: int = 64) -> None:
        if n_pages <= 0 or page_size < 16 or page_size > 4096 or page_size & (page_size - 1):
            raise ValueError(f"pages must hold a power of two of tokens, 16 to 4096, got {n_pages} of {page_size}")
        if n_pages * page_size >= 1 << 31:
            raise ValueError(f"{n_pages} pages of {page_size} tokens: their slots pass 32 bits")
        self.n_pages, self.page_size = int(n_pages), int(page_size)
        self.max_keys: int | None = None  # that a sequence may hold
        self._free = list(range(self.n_pages - 1, -1, -1))  # taken from the end: low pages first
        self._holders = np.zeros(self.n_pages, np.int32)    # sequences that hold the page
        self._pages = np.zeros((8, 8), np.int32)            # [sequence][page of it]
        self._lengths = np.full(8, -1, np.int64)            # tokens; -1: no sequence
        self._evicted = np.zeros(8, np.int64)               # tokens before them whose keys have left
        self._firsts = np.full(8, _ALL, np.int64)           # tokens at the start whose keys are still at their places

    def _held(self, n_tokens):
        return -(-n_tokens // self.page_size)

    def _check(self, seqs) -> np.ndarray:
        at = np.asarray(seqs)
        if at.ndim != 1 or at.size == 0 or at.dtype.kind not in "iu":
            raise ValueError(f"a list of sequences is needed, got {seqs!r}")
        at = at.astype(np.int64)
        gone = (at < 0) | (at >= len(self._lengths))
        if gone.any() or (self._lengths[at] < 0).any():
            raise KeyError(f"no such sequence among {at.tolist()}")
        if np.unique(at).size != at.size:
            raise ValueError(f"the same sequence twice in {at.tolist()}")
        return at

    def _room(self, need: int) -> None:
        if need > len(self._free):
            raise RuntimeError(f"the cache's {self.n_pages} pages are taken: {need} needed, {len(self._free)} free")

    def _widen(self, width: int) -> None:
        """Space for sequences of ``width`` pages."""
        if width > self._pages.shape[1]:
            wider = np.zeros((self._pages.shape[0], max(width, 2 * self._pages.shape[1])), np.int32)
            wider[:, :self._pages.shape[1]] = self._pages
            self._pages = wider

    def _take(self, seq: int, count: int) -> None:
        """`count` more pages behind those that the sequence's length fills; there is space for them."""
        at = int(self._held(self._lengths[seq]))
        new = self._free[-count:][::-1]
        del self._free[-count:]
        self._pages[seq, at:at + count] = new
        self._holders[new] = 1

    def add(self) -> int:
        """A new sequence without tokens."""
        free = np.flatnonzero(self._lengths < 0)
        if free.size == 0:
            free = np.array([len(self._lengths)])
            self._lengths = np.concatenate((self._lengths, np.full(len(self._lengths), -1, np.int64)))
            self._pages = np.concatenate((self._pages, np.zeros_like(self._pages)))
            self._evicted = np.concatenate((self._evicted, np.zeros_like(self._evicted)))
            self._firsts = np.concatenate((self._firsts, np.full_like(self._firsts, _ALL)))
        self._lengths[free[0]] = self._evicted[free[0]] = 0
        self._firsts[free[0]] = _ALL
        return int(free[0])

    def length(self, seq: int) -> int:
        return int(self._lengths[self._check([seq])[0]])

    def pages(self, seq: int) -> list[int]:
        at = self._check([seq])[0]
        return self._pages[at, :self._held(self._lengths[at])].tolist()

    def fork(self, seq: int, count: int = 1) -> tuple[list[int], list[int], list[int]]:
        """``count`` new sequences with ``seq``'s tokens, and the page moves (sources, destinations) that they need."""
        parent = int(self._check([seq])[0])
        if count < 0:
            raise ValueError(f"a fork into {count} sequences")
        n = int(self._lengths[parent])
        full, part = n // self.page_size, n % self.page_size > 0
        self._room(count * part)
        children, src, dst = [], [], []
        for _ in range(count):
            child = self.add()
            self._pages[child, :full] = self._pages[parent, :full]
            self._holders[self._pages[parent, :full]] += 1
            self._lengths[child] = full * self.page_size
            if part:
                self._take(child, 1)
                src.append(int(self._pages[parent, full]))
                dst.append(int(self._pages[child, full]))
            self._lengths[child], self._evicted[child], self._firsts[child] = n, self._evicted[parent], self._firsts[parent]
            children.append(child)
        return children, src, dst

    def free(self, seq: int) -> None:
        at = int(self._check([seq])[0])
        held = self._pages[at, :self._held(self._lengths[at])]
        self._holders[held] -= 1
        self._free.extend(held[self._holders[held] == 0][::-1].tolist())
        self._lengths[at] = -1

    def extend(self, seqs, counts=1) -> dict:
        """``counts`` (a number or one a sequence) more tokens of each of ``seqs``, all or none.  int32 arrays for a
        batch of these tokens, sequence by sequence: ``positions`` and ``slots`` of the tokens, ``starts`` of the
        sequences' runs, ``prefix`` (full pages that all share, in front), and for every token the pages behind them
        (``tables``) and the tokens in those up to itself (``lengths``).  ``fresh``: no sequence had tokens, and what
        tells of earlier ones is empty.  Of the sequences: ``seqs``, ``counts``, ``keys`` with the new
        ones, ``pages`` and ``firsts``, the tokens at their starts that evictions have left in place."""
        at = self._check(seqs)
        counts = np.broadcast_to(np.asarray(counts), at.shape)
        if counts.dtype.kind not in "iu" or (counts <= 0).any():
            raise ValueError(f"token counts must be positive, got {counts.tolist()}")
        counts = counts.astype(np.int64)
        before = self._lengths[at]  # a copy
        after = before + counts
        longest = int((after + self._evicted[at]).max())
        if longest >= 1 << 29:
            raise ValueError(f"sequences must stay below 2^29 tokens, got {longest}")
        if self.max_keys is not None and after.max() > self.max_keys:
            raise RuntimeError(f"the cache keeps the weights of {self.max_keys} keys a sequence, {int(after.max())} needed")
        need = self._held(after) - self._held(before)
        self._room(int(need.sum()))
        self._widen(int(self._held(after.max())))
        for s in np.flatnonzero(need):
            self._take(int(at[s]), int(need[s]))
        self._lengths[at] = after
        try:
            return self._batch(at, before, after, counts)
        except BaseException:  # no memory for the arrays
            self.undo_extend(at, counts)
            raise

    def undo_extend(self, seqs, counts) -> None:
        """Takes back the extension of ``seqs`` by ``counts`` that was made last."""
        for s, n in zip(np.asarray(seqs)[::-1], np.asarray(counts)[::-1]):
            before, after = int(self._lengths[s]) - int(n), int(self._lengths[s])
            pages = self._pages[s, self._held(before):self._held(after)]
            self._holders[pages] = 0
            self._free.extend(pages[::-1].tolist())
            self._lengths[s] = before

    def _batch(self, at, before, after, counts) -> dict:
        """extend's arrays, of the tokens from ``before`` up to ``after`` of the sequences."""
        starts = np.concatenate(([0], np.cumsum(counts)))
        row = np.repeat(np.arange(at.size), counts)
        positions = np.arange(starts[-1]) - starts[row] + before[row]
        held = self._held(after)
        pages = self._pages[at, :int(held.max())]  # a copy
        if held.min() < pages.shape[1]:
            pages[np.arange(pages.shape[1]) >= held[:, None]] = -1
        slots = pages[row, positions // self.page_size].astype(np.int64) * self.page_size + positions % self.page_size
        of = dict(seqs=at, counts=counts, keys=after, pages=pages, firsts=self._firsts[at])
        if not before.any():  # prompts, which attend to themselves
            none = np.zeros(0, np.int32)
            out = dict(positions=positions, slots=slots, starts=starts, prefix=none, tables=none.reshape(0, 0), lengths=none, **of)
            return {**{k: v.astype(np.int32) for k, v in out.items()}, "fresh": True}
        full = int(before.min()) // self.page_size
        same = (pages[:, :full] == pages[:1, :full]).all(axis=0)
        shared = full if same.all() else int(np.argmin(same))
        out = dict(positions=positions + self._evicted[at][row], slots=slots, starts=starts, prefix=pages[0, :shared],
                   tables=pages[row, shared:], lengths=positions + 1 - shared * self.page_size, **of)
        return {**{k: v.astype(np.int32) for k, v in out.items()}, "fresh": False}

    def eviction(self, seqs, keep: int) -> dict:
        """What cutting those of ``seqs`` with more than ``keep`` keys to as many needs, for ``evict`` afterwards: the cut
        ones (``seqs``), their ``keys`` and ``pages``, and the moves (``src``, ``dst``) to free pages of those to be written
        that others hold too, which ``pages`` has already."""
        at = self._check(seqs)
        if keep <= 0:
            raise ValueError(f"a cut to {keep} keys")
        at = at[self._lengths[at] > keep]
        holders, free = self._holders.copy(), list(self._free)
        width = self._held(int(self._lengths[at].max())) if at.size else 0
        pages = self._pages[at, :width].copy()
        src, dst = [], []
        for row in range(at.size):
            for i in range(self._held(keep)):
                page = int(pages[row, i])
                if holders[page] > 1:
                    if not free:
                        raise RuntimeError(f"the cache's {self.n_pages} pages are taken: no page for a shared one to be cut")
                    holders[page] -= 1
                    src.append(page)
                    dst.append(free.pop())
                    pages[row, i] = dst[-1]
        pages = np.where(np.arange(width) < self._held(self._lengths[at])[:, None], pages, -1).astype(np.int32)
        return dict(seqs=at, keys=self._lengths[at].astype(np.int32), pages=pages, src=src, dst=dst)

    def evict(self, plan: dict, keep: int, first: int = 0) -> None:
        """Books the ``eviction`` that was asked for last, which leaves the ``first`` keys in place."""
        del self._free[len(self._free) - len(plan["dst"]):]
        self._holders[plan["dst"]] = 1
        np.subtract.at(self._holders, plan["src"], 1)
        for s, n, pages in zip(plan["seqs"], plan["keys"], plan["pages"]):
            held = self._held(int(n))
            self._pages[s, :held] = pages[:held]
            left = pages[self._held(keep):held]
            self._holders[left] -= 1
            self._free.extend(left[self._holders[left] == 0][::-1].tolist())
            self._lengths[s] = keep
            self._evicted[s] += int(n) - keep
            self._firsts[s] = min(self._firsts[s], first)

    def moves(self) -> tuple[list[int], list[int]]:
        """The page moves (sources, destinations) of a compaction: pages that are held go to the front."""
        held = np.flatnonzero(self._holders)
        dst = np.flatnonzero(self._holders[:held.size] == 0)
        return held[held >= held.size].tolist(), dst.tolist()

    def compact(self) -> tuple[list[int], list[int]]:
        """Moves pages to the front, so that those held are the first: the moves (sources, destinations)."""
        src, dst = self.moves()
        if src:
            to = np.arange(self.n_pages, dtype=np.int32)
            to[src] = dst
            self._pages = to[self._pages]
            self._holders[dst] = self._holders[src]
            self._holders[src] = 0
        self._free = list(range(self.n_pages - 1, np.count_nonzero(self._holders) - 1, -1))
        return src, dst

    def stats(self) -> dict:
        live = self._lengths >= 0
        return {"pages": self.n_pages, "page_size": self.page_size, "free_pages": len(self._free),
                "shared_pages": int((self._holders > 1).sum()), "sequences": int(live.sum()),
                "tokens": int(self._lengths[live].sum())}


@dataclass
class PagedBatch:
    """Tokens to be run through the layers, on the device: see PageTable.extend.  Row i of the activations is token i;
    ``starts[1:] - 1`` are the sequences' last ones."""
    positions: torch.Tensor      # int32 [tokens]
    slots: torch.Tensor          # int32 [tokens]
    starts: torch.Tensor         # int32 [sequences + 1]
    tables: torch.Tensor         # int32 [tokens, pages], of a fresh batch empty
    lengths: torch.Tensor        # int32 [tokens], of a fresh batch empty
    prefix_table: torch.Tensor   # int32 [pages]
    prefix_len: int
    fresh: bool                  # whole prompts: no sequence had tokens
    tokens: int
    end: int                     # past the largest position
    host: dict = field(default_factory=dict, repr=False)  # of the sequences: see PageTable.extend
    _made: dict = field(default_factory=dict, repr=False)

    def sequences(self) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """Of each sequence its pages (int32 ``[sequences, pages]``), its keys and its number, on the device: what layers by
        sequences read, and captured ones read again at every replay."""
        def make():
            if self.positions.is_cuda and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("a batch's arrays cannot be copied while a graph is captured: call sequences() and plan() before")
            made = _to_device([self.host[n] for n in ("pages", "keys", "seqs")], self.positions.device)
            return made, made
        return self._once("sequences", make)

    def plan(self, config: AttentionConfig, window: int | None, first: int, key_weights: bool = True) -> ops.AttentionPlan:
        """The division of its tokens' attention over the cache, for all layers with this window; without ``key_weights``
        for those of a cache that keeps none."""
        key = (config.num_heads, config.num_kv_heads, config.head_dim, window, first, key_weights)
        if not key_weights and (*key[:5], True) in self._made:  # made for more: as good
            key = (*key[:5], True)

        def make():
            made = ops.attention_plan(self.host["counts"], self.host["keys"], *key[:5], self.positions.device, key_weights)
            return made, (made.data,)
        return self._once(key, make)

    def _once(self, key, make):
        """``make()``'s first part, made at the first call; its second are the device tensors in it.  Calls on other streams
        than the first one's wait there for the copies, but for captured ones: a graph's replays come behind them anyway,
        since torch.cuda.graph waits for the device before it captures."""
        device = self.positions.device
        made = self._made.get(key)
        if made is None:
            what, tensors = make()
            event = torch.cuda.current_stream(device).record_event() if device.type == "cuda" else None
            self._made[key] = made = (what, tensors, _stream(device), event)
        elif made[2] != _stream(device) and not torch.cuda.is_current_stream_capturing():
            stream = torch.cuda.current_stream(device)
            stream.wait_event(made[3])
            for t in made[1]:
                t.record_stream(stream)
        return made[0]


def _stream(device: torch.device) -> int | None:
    """The current stream's number, None on the CPU."""
    return torch._C._cuda_getCurrentRawStream(device.index) if device.type == "cuda" else None


def _to_device(parts: list, device: torch.device) -> tuple:
    """int32 arrays in one copy."""
    host = torch.empty(sum(x.size for x in parts), dtype=torch.int32, pin_memory=device.type == "cuda")
    np.concatenate([x.ravel() for x in parts], out=host.numpy())
    return tuple(t.view(x.shape) for t, x in zip(host.to(device, non_blocking=True).split([x.size for x in parts]), parts))


class PagedKVCache:
    """Keys and values of ``n_layers`` layers for many sequences: ``pool [2 * n_layers, n_pages, page_size, n_kv,
    head_dim]`` of the ``precision`` ("fp16" or "bf16", as DeviceKVCache's), a layer's keys, then its values.  With
    ``weighted`` = (sequences, keys) also the float32 ``weights [n_layers, sequences, n_kv, keys]`` that each key was given
    so far by the tokens behind it, for ``evict``; it then holds at most as many sequences, each of at most as many keys."""

    def __init__(self, device: torch.device | str, n_layers: int, n_kv: int, head_dim: int, n_pages: int,
                 page_size: int = 64, precision: str = "fp16", weighted: tuple[int, int] | None = None) -> None:
        if precision not in _KV_DTYPES:
            raise ValueError(f"unsupported KV cache precision for the device cache: {precision}")
        if n_layers <= 0 or n_kv <= 0 or head_dim <= 0:
            raise ValueError(f"a cache of {n_layers} layers of {n_kv} heads of {head_dim}")
        self.table = PageTable(n_pages, page_size)
        self.precision = precision
        self.dtype = _KV_DTYPES[precision][0]
        self.pool = torch.empty((2 * n_layers, n_pages, page_size, n_kv, head_dim), dtype=self.dtype, device=device)
        self.device = self.pool.device  # "cuda" is the current device now, not the one of a later call
        self.first_tokens = 0  # that a layer saw beside its window, the most so far
        self.weights = None
        if weighted is not None:
            weighted = tuple(operator.index(x) for x in weighted)
            if len(weighted) != 2 or min(weighted) <= 0:
                raise ValueError(f"weights of (sequences, keys), got {weighted}")
            self.table.max_keys = weighted[1]
            self.weights = torch.zeros((n_layers, weighted[0], n_kv, weighted[1]), dtype=torch.float32, device=self.device)

    def layer(self, layer_idx: int) -> tuple[torch.Tensor, torch.Tensor]:
        """The layer's key and value pages ``[n_pages, page_size, n_kv, head_dim]``."""
        if not 0 <= layer_idx < self.pool.shape[0] // 2:
            raise IndexError(f"layer {layer_idx} of {self.pool.shape[0] // 2}")
        return self.pool[2 * layer_idx], self.pool[2 * layer_idx + 1]

    def add(self) -> int:
        """A new sequence without tokens."""
        seq = self.table.add()
        if self.weights is not None and seq >= self.weights.shape[1]:
            self.table.free(seq)
            raise RuntimeError(f"the cache keeps the weights of {self.weights.shape[1]} sequences, which are taken")
        return seq

    def length(self, seq: int) -> int:
        """The tokens whose keys it holds."""
        return self.table.length(seq)

    def fork(self, seq: int, count: int = 1) -> list[int]:
        """New sequences with ``seq``'s tokens, which share its full pages."""
        children, src, dst = self.table.fork(seq, count)
        try:
            if self.weights is not None:
                if max(children, default=0) >= self.weights.shape[1]:
                    raise RuntimeError(f"the cache keeps the weights of {self.weights.shape[1]} sequences, which are taken")
                n = self.table.length(seq)
                for child in children:
                    self.weights[:, child, :, :n].copy_(self.weights[:, seq, :, :n])
            if src:
                ops.copy_pages(self.pool, src, dst)
        except BaseException:  # sequences without their last page must not stay
            for child in reversed(children):
                self.table.free(child)
            raise
        return children

    def free(self, seq: int) -> None:
        self.table.free(seq)

    def evict(self, seqs, keep: int, recent: int = 0, first: int = 0) -> list[int]:
        """Cuts those of ``seqs`` with more than ``keep`` keys to as many, in every layer and KV head by itself: the
        ``first`` and the last ``recent`` ones stay, and of the others those of the largest weights (ops.evict_keys).
        Returns the sequences that were cut.  Pages of the kept part that others hold too are copied first, to free ones:
        RuntimeError, and nothing done, where there are too few of them, though the cut itself might free others (its keys
        move within the pages, which are read to its end).  New tokens go on at their positions in the whole text.  A
        window counts keys that are held: layers with one need ``recent`` of at least it.  What layers see beside one are
        the keys at the start: a ``first`` below their ``first_tokens`` is refused, and so is such a layer on a sequence
        that was cut with one before.  Batches made before are void."""
        if self.weights is None:
            raise ValueError("a cache without weights: give `weighted` when it is made")
        keep, recent, first = operator.index(keep), operator.index(recent), operator.index(first)
        if recent < 0 or first < 0 or recent + first > keep:
            raise ValueError(f"{keep} keys kept, of them the first {first} and the last {recent}")
        if first < self.first_tokens:
            raise ValueError(f"the first {first} keys kept, of {self.first_tokens} that layers see beside their windows")
        plan = self.table.eviction(seqs, keep)
        if plan["seqs"].size:
            tables, lengths, rows = _to_device([plan["pages"], plan["keys"], plan["seqs"].astype(np.int32)], self.device)
            if plan["src"]:
                ops.copy_pages(self.pool, plan["src"], plan["dst"])
            ops.evict_keys(self.pool, self.weights, tables, lengths, rows, keep, recent=recent, first=first)
            self.table.evict(plan, keep, first)  # once the work is under way
        return plan["seqs"].tolist()

    def compact(self) -> int:
        """Moves the held pages to the pool's front and returns how many they are.  Batches made before are void."""
        src, dst = self.table.moves()
        if src:
            ops.copy_pages(self.pool, src, dst)
        self.table.compact()  # once the copies are under way: the pages they came from are as they were
        return self.table.n_pages - self.table.stats()["free_pages"]

    def extend(self, seqs, counts=1) -> PagedBatch:
        """Room for ``counts`` (a number or one a sequence) more tokens of each sequence, and their batch.  Every layer
        has to run it before the sequences are extended, forked, freed, evicted from or compacted again.  Prompts do
        better in a batch of their own."""
        x = self.table.extend(seqs, counts)
        try:
            return self._to_device(x)
        except BaseException:  # no memory for the arrays
            self.table.undo_extend(seqs, np.diff(x["starts"]))
            raise

    def _to_device(self, x: dict) -> PagedBatch:
        names = ("positions", "slots", "starts", "lengths", "prefix", "tables")
        d = dict(zip(names, _to_device([x[n] for n in names], self.device)))
        return PagedBatch(d["positions"], d["slots"], d["starts"], d["tables"], d["lengths"], d["prefix"],
                          x["prefix"].size * self.table.page_size, x["fresh"], x["positions"].size,
                          int(x["positions"].max()) + 1,
                          {**{n: x[n] for n in ("seqs", "counts", "keys", "pages")}, "first": int(x["firsts"].min())})

    def stats(self) -> dict:
        return {**self.table.stats(), "resident_bytes": self.pool.numel() * self.pool.element_size(),
                "device": str(self.device), "precision": self.precision}


class BatchedAttention:
    """StreamedAttention's layer for a PagedBatch (inference: no gradients).  Refuses models whose steps batch_attention
    does not take, though it could run their prompts: groups of more than 32 query heads.  ``first_tokens`` at the start
    of a sequence stay visible beside the windows of layers that have one.  Where a layer's tensors hold
    ``q_norm.weight`` or ``k_norm.weight [head_dim]``, its queries' or keys' heads are normalised before they are rotated
    (``config.rms_norm_eps``); a projection without a bias tensor has none."""

    def __init__(self, config: AttentionConfig, first_tokens: int = 0) -> None:
        heads, kv, dim = config.num_heads, config.num_kv_heads, config.head_dim
        if kv <= 0 or heads <= 0 or heads % kv or heads // kv > 32 or heads > 4096:
            raise ValueError(f"{heads} query heads over {kv} KV heads (groups of 1 to 32, up to 4096 heads)")
        if dim < 8 or dim % 8 or dim > 128:
            raise ValueError(f"head size {dim} (8 to 128, a multiple of 8)")
        first_tokens = operator.index(first_tokens)
        if first_tokens < 0:
            raise ValueError(f"{first_tokens} first tokens")
        self.config = config
        self.first_tokens = first_tokens
        self._tables: dict = {}  # device -> (cos, sin) of the positions so far
        self._kept: list = []    # smaller ones, which captured graphs may still read

    def rope_tables(self, n_positions: int, device: torch.device) -> tuple[torch.Tensor, torch.Tensor]:
        """bfloat16 ``[n, head_dim / 2]`` cosines and sines, row p as rope_cos_sin's of position p, n >= n_positions."""
        held = self._tables.get(device)
        if held is None or held[0].shape[0] < n_positions:
            n = max(1024, 1 << (int(n_positions) - 1).bit_length())
            angle = torch.arange(n, dtype=torch.float32, device=device)[:, None] * yarn_inv_freq(self.config, device).float()
            s = yarn_attention_scaling(self.config)
            held = ((torch.cos(angle) * s).to(torch.bfloat16), (torch.sin(angle) * s).to(torch.bfloat16))
            torch.cuda.current_stream(device).synchronize()  # any stream may read them from here on
            self._kept.append(self._tables.get(device))
            self._tables[device] = held
        return held

    @staticmethod
    def _suffixes(batch: PagedBatch, window: int | None) -> bool:
        """Whether a batch with tokens behind cached ones goes by sequences rather than row by row: if any has several.
        Short suffixes behind a long prefix that all share do better by rows, for which it is read once (64 heads over
        8 of size 64, us by rows and by sequences: 64 behind 8,192 tokens 2 each 49 and 85, 8 each 159 and 126; 8 behind
        8,192 2 each 18 and 26; 200 behind 1,000 2 each 38 and 42).  The prefix's length itself is no part of the rule,
        which costs a few us where it is short and the sequences are few (66 behind 960 2 each 23 and 20).  A captured
        graph, which may be replayed with other ``tables`` and ``lengths`` of the rows, keeps to them."""
        count = batch.starts.shape[0] - 1
        if batch.tokens == count or not batch.host or torch.cuda.is_current_stream_capturing():
            return False
        if window is None and batch.tokens <= 4 * count and 8 * batch.prefix_len >= 7 * batch.host["keys"].max():
            return False
        return True

    def forward(self, layer_idx: int, hidden: torch.Tensor, tensors: dict, batch: PagedBatch, kv_cache: PagedKVCache,
                sliding_window: int | None = None) -> torch.Tensor:
        """bfloat16 ``hidden [tokens, hidden_size]`` of the batch's tokens -> the layer's output for them; their keys
        and values are stored to the cache.  ``tensors`` and ``sliding_window`` (0: no window) as
        StreamedAttention.forward's."""
        cfg = self.config
        prefix = f"model.layers.{layer_idx}.self_attn"
        if hidden.dim() != 2 or hidden.shape[0] != batch.tokens:
            raise ValueError(f"a batch of {batch.tokens} tokens, got hidden {tuple(hidden.shape)}")
        window = (sliding_window if sliding_window is not None else cfg.sliding_window) or None  # 0: none
        first = self.first_tokens if window else 0
        if first:
            if batch.host.get("first", first) < first:
                raise ValueError(f"{first} first tokens beside a window, of sequences that were cut to the first {batch.host['first']} keys")
            kv_cache.first_tokens = max(kv_cache.first_tokens, first)
        lin = torch.nn.functional.linear

        def project(name: str, heads: int) -> torch.Tensor:
            x = lin(hidden, tensors[f"{prefix}.{name}.weight"], tensors.get(f"{prefix}.{name}.bias"))
            return x.view(batch.tokens, heads, cfg.head_dim)

        q, k, v = project("q_proj", cfg.num_heads), project("k_proj", cfg.num_kv_heads), project("v_proj", cfg.num_kv_heads)
        weights = kv_cache.weights
        chunks = weights is not None or first > 0 or (not batch.fresh and self._suffixes(batch, window))
        if chunks:  # before the keys are stored: what cannot be planned leaves the cache as it was
            tables, lengths, rows = batch.sequences()
            plan = batch.plan(cfg, window, first, weights is not None)
        k_pages, v_pages = kv_cache.layer(layer_idx)
        cos, sin = self.rope_tables(batch.end, q.device)
        norms = [tensors.get(f"{prefix}.{name}.weight") for name in ("q_norm", "k_norm")]
        norms = [t if t is None else t.to(torch.bfloat16).contiguous() for t in norms]
        q, k = ops.paged_append(q, k, v, cos, sin, batch.positions, batch.slots, k_pages, v_pages,
                                want_keys=batch.fresh and not chunks, q_norm=norms[0], k_norm=norms[1], eps=cfg.rms_norm_eps)
        sinks = tensors.get(f"{prefix}.sinks")
        if sinks is not None:
            sinks = sinks.to(torch.bfloat16).contiguous()
        if chunks:
            if weights is None:
                context = ops.chunk_attention(q, k_pages, v_pages, tables, lengths, plan, sinks)
            else:
                context, lse = ops.chunk_attention(q, k_pages, v_pages, tables, lengths, plan, sinks, want_lse=True)
                ops.add_key_weights(q, lse, k_pages, tables, lengths, plan, weights[layer_idx], rows)
        elif batch.fresh:
            context = ops.prompt_attention(q, k, v, batch.starts, sinks, window)
        else:
            context = torch.empty_like(q)
            for i in range(0, batch.tokens, _MAX_ROWS):
                rows = slice(i, i + _MAX_ROWS)
                ops.batch_attention(q[rows], k_pages, v_pages, batch.tables[rows], batch.lengths[rows],
                                    batch.prefix_table, batch.prefix_len, sinks, window, out=context[rows])
        o_weight = tensors[f"{prefix}.o_proj.weight"]
        return lin(context.view(batch.tokens, -1).to(o_weight.dtype), o_weight, tensors.get(f"{prefix}.o_proj.bias"))
