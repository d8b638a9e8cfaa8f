"""A KV cache of many sequences in pages, and the attention layer over it.

``PageTable``         which sequence holds which pages: host bookkeeping alone.
``PagedKVCache``      a PageTable with its pages in HBM, one slab for all
                      layers' keys and values, so that a fork or a compaction
                      is one launch (ops.copy_pages) whatever the number of
                      layers.
``BatchedAttention``  StreamedAttention's layer (projections, RoPE, sinks,
                      window) for a batch of tokens of several sequences:
                      whole prompts by ops.prompt_attention, tokens behind
                      cached ones by ops.batch_attention, each token a row
                      of it.  Pages that all of the batch's sequences share
                      are read once on layers without a window, if they are
                      many.

Pages are shared while they are full and never written then: a fork takes its
parent's full pages as they are and a copy of the last one.  Work on the cache
is ordered by the stream it runs on; a caller with several streams orders them.
"""

from __future__ import annotations

from dataclasses import dataclass

import numpy as np
import torch

from . import ops
from .attention import _KV_DTYPES, AttentionConfig, yarn_attention_scaling, yarn_inv_freq


_MAX_ROWS = 65535  # of a batch_attention call


class PageTable:
    """Pages of ``page_size`` tokens among sequences, numbered as they were added (numbers are used again)."""

    def __init__(self, n_pages: int, page_size: int = 64) -> None:
        if n_pages <= 0 or page_size < 16 or page_size > 4096 or page_size & (page_size - 1):
            raise ValueError(f"pages must hold a power of two of tokens, 16 to 4096, got {n_pages} of {page_size}")
        if n_pages * page_size >= 1 << 31:
            raise ValueError(f"{n_pages} pages of {page_size} tokens: their slots pass 32 bits")
        self.n_pages, self.page_size = int(n_pages), int(page_size)
        self._free = list(range(self.n_pages - 1, -1, -1))  # taken from the end: low pages first
        self._holders = np.zeros(self.n_pages, np.int32)    # sequences that hold the page
        self._pages = np.zeros((8, 8), np.int32)            # [sequence][page of it]
        self._lengths = np.full(8, -1, np.int64)            # tokens; -1: no sequence

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
        self._lengths[free[0]] = 0
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
            self._lengths[child] = n
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
        tells of earlier ones is empty."""
        at = self._check(seqs)
        counts = np.broadcast_to(np.asarray(counts), at.shape)
        if counts.dtype.kind not in "iu" or (counts <= 0).any():
            raise ValueError(f"token counts must be positive, got {counts.tolist()}")
        counts = counts.astype(np.int64)
        before = self._lengths[at]  # a copy
        after = before + counts
        if after.max() >= 1 << 29:
            raise ValueError(f"sequences must stay below 2^29 tokens, got {int(after.max())}")
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
        slots = self._pages[at[row], positions // self.page_size].astype(np.int64) * self.page_size + positions % self.page_size
        if not before.any():  # prompts, which attend to themselves
            none = np.zeros(0, np.int32)
            out = dict(positions=positions, slots=slots, starts=starts, prefix=none, tables=none.reshape(0, 0), lengths=none)
            return {**{k: v.astype(np.int32) for k, v in out.items()}, "fresh": True}
        full = int(before.min()) // self.page_size
        rows = self._pages[at, :full]
        same = (rows == rows[:1]).all(axis=0)
        shared = full if same.all() else int(np.argmin(same))
        tables = self._pages[at, shared:self._held(int(after.max()))]
        tables = np.where(np.arange(tables.shape[1]) < (self._held(after) - shared)[:, None], tables, -1)
        out = dict(positions=positions, slots=slots, starts=starts, prefix=self._pages[at[0], :shared], tables=tables[row],
                   lengths=positions + 1 - shared * self.page_size)
        return {**{k: v.astype(np.int32) for k, v in out.items()}, "fresh": False}

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


class PagedKVCache:
    """Keys and values of ``n_layers`` layers for many sequences: ``pool [2 * n_layers, n_pages, page_size, n_kv,
    head_dim]`` of the ``precision`` ("fp16" or "bf16", as DeviceKVCache's), a layer's keys, then its values."""

    def __init__(self, device: torch.device | str, n_layers: int, n_kv: int, head_dim: int, n_pages: int,
                 page_size: int = 64, precision: str = "fp16") -> None:
        if precision not in _KV_DTYPES:
            raise ValueError(f"unsupported KV cache precision for the device cache: {precision}")
        if n_layers <= 0 or n_kv <= 0 or head_dim <= 0:
            raise ValueError(f"a cache of {n_layers} layers of {n_kv} heads of {head_dim}")
        self.table = PageTable(n_pages, page_size)
        self.precision = precision
        self.dtype = _KV_DTYPES[precision][0]
        self.pool = torch.empty((2 * n_layers, n_pages, page_size, n_kv, head_dim), dtype=self.dtype, device=device)
        self.device = self.pool.device  # "cuda" is the current device now, not the one of a later call

    def layer(self, layer_idx: int) -> tuple[torch.Tensor, torch.Tensor]:
        """The layer's key and value pages ``[n_pages, page_size, n_kv, head_dim]``."""
        if not 0 <= layer_idx < self.pool.shape[0] // 2:
            raise IndexError(f"layer {layer_idx} of {self.pool.shape[0] // 2}")
        return self.pool[2 * layer_idx], self.pool[2 * layer_idx + 1]

    def add(self) -> int:
        """A new sequence without tokens."""
        return self.table.add()

    def length(self, seq: int) -> int:
        return self.table.length(seq)

    def fork(self, seq: int, count: int = 1) -> list[int]:
        """New sequences with ``seq``'s tokens, which share its full pages."""
        children, src, dst = self.table.fork(seq, count)
        try:
            if src:
                ops.copy_pages(self.pool, src, dst)
        except BaseException:  # sequences without their last page must not stay
            for child in reversed(children):
                self.table.free(child)
            raise
        return children

    def free(self, seq: int) -> None:
        self.table.free(seq)

    def compact(self) -> int:
        """Moves the held pages to the pool's front and returns how many they are.  Batches made before are void."""
        src, dst = self.table.moves()
        if src:
            ops.copy_pages(self.pool, src, dst)
        self.table.compact()  # once the copies are under way: the pages they came from are as they were
        return self.table.n_pages - self.table.stats()["free_pages"]

    def extend(self, seqs, counts=1) -> PagedBatch:
        """Room for ``counts`` (a number or one a sequence) more tokens of each sequence, and their batch.  Every layer
        has to run it before the sequences are extended, forked, freed or compacted again.  A batch in which any
        sequence has tokens goes row by row: prompts do better in a batch of their own."""
        x = self.table.extend(seqs, counts)
        try:
            return self._to_device(x)
        except BaseException:  # no memory for the arrays
            self.table.undo_extend(seqs, np.diff(x["starts"]))
            raise

    def _to_device(self, x: dict) -> PagedBatch:
        names = ("positions", "slots", "starts", "lengths", "prefix", "tables")
        host = torch.empty(sum(x[n].size for n in names), dtype=torch.int32, pin_memory=self.device.type == "cuda")
        np.concatenate([x[n].ravel() for n in names], out=host.numpy())
        parts = host.to(self.device, non_blocking=True).split([x[n].size for n in names])
        d = {n: p.view(x[n].shape) for n, p in zip(names, parts)}
        return PagedBatch(d["positions"], d["slots"], d["starts"], d["tables"], d["lengths"], d["prefix"],
                          x["prefix"].size * self.table.page_size, x["fresh"], x["positions"].size,
                          int(x["positions"].max()) + 1)

    def stats(self) -> dict:
        return {**self.table.stats(), "resident_bytes": self.pool.numel() * self.pool.element_size(),
                "device": str(self.device), "precision": self.precision}


class BatchedAttention:
    """StreamedAttention's layer for a PagedBatch (inference: no gradients).  Refuses models whose steps batch_attention
    does not take, though it could run their prompts: groups of more than 32 query heads."""

    def __init__(self, config: AttentionConfig) -> None:
        heads, kv, dim = config.num_heads, config.num_kv_heads, config.head_dim
        if kv <= 0 or heads <= 0 or heads % kv or heads // kv > 32 or heads > 4096:
            raise ValueError(f"{heads} query heads over {kv} KV heads (groups of 1 to 32, up to 4096 heads)")
        if dim < 8 or dim % 8 or dim > 128:
            raise ValueError(f"head size {dim} (8 to 128, a multiple of 8)")
        self.config = config
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

    def forward(self, layer_idx: int, hidden: torch.Tensor, tensors: dict, batch: PagedBatch, kv_cache: PagedKVCache,
                sliding_window: int | None = None) -> torch.Tensor:
        """bfloat16 ``hidden [tokens, hidden_size]`` of the batch's tokens -> the layer's output for them; their keys
        and values are stored to the cache.  ``tensors`` and ``sliding_window`` (0: no window) as
        StreamedAttention.forward's."""
        cfg = self.config
        prefix = f"model.layers.{layer_idx}.self_attn"
        if hidden.dim() != 2 or hidden.shape[0] != batch.tokens:
            raise ValueError(f"a batch of {batch.tokens} tokens, got hidden {tuple(hidden.shape)}")
        lin = torch.nn.functional.linear

        def project(name: str, heads: int) -> torch.Tensor:
            x = lin(hidden, tensors[f"{prefix}.{name}.weight"], tensors[f"{prefix}.{name}.bias"])
            return x.view(batch.tokens, heads, cfg.head_dim)

        q, k, v = project("q_proj", cfg.num_heads), project("k_proj", cfg.num_kv_heads), project("v_proj", cfg.num_kv_heads)
        k_pages, v_pages = kv_cache.layer(layer_idx)
        cos, sin = self.rope_tables(batch.end, q.device)
        q, k = ops.paged_append(q, k, v, cos, sin, batch.positions, batch.slots, k_pages, v_pages, want_keys=batch.fresh)
        window = (sliding_window if sliding_window is not None else cfg.sliding_window) or None  # 0: none
        sinks = tensors.get(f"{prefix}.sinks")
        if sinks is not None:
            sinks = sinks.to(torch.bfloat16).contiguous()
        if batch.fresh:
            context = ops.prompt_attention(q, k, v, batch.starts, sinks, window)
        else:
            context = torch.empty_like(q)
            for i in range(0, batch.tokens, _MAX_ROWS):
                rows = slice(i, i + _MAX_ROWS)
                ops.batch_attention(q[rows], k_pages, v_pages, batch.tables[rows], batch.lengths[rows],
                                    batch.prefix_table, batch.prefix_len, sinks, window, out=context[rows])
        o_weight = tensors[f"{prefix}.o_proj.weight"]
        return lin(context.view(batch.tokens, -1).to(o_weight.dtype), o_weight, tensors[f"{prefix}.o_proj.bias"])
