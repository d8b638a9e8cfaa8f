"""The host's division of chunk attention, and what the C entry points of long conversations refuse before any device
work (no GPU)."""

from __future__ import annotations

import random
import struct

import numpy as np
import pytest

from klcquant_amd import _native as nat
from klcquant_amd import ops


def plan(counts, lengths, heads=64, kv=8, dim=64, window=0, first=0, capacity=1 << 18):
    counts, lengths = np.array(counts, np.int32), np.array(lengths, np.int32)
    sizes, out = np.zeros(12, np.int64), np.full(capacity, -7, np.int32)
    nat.call("klc_attn_plan", counts.ctypes.data, lengths.ctypes.data, len(counts), heads, kv, dim, window, first,
             out.ctypes.data if capacity else None, capacity, sizes.ctypes.data)
    return sizes.tolist(), out


def sees(pos, key, window, first):
    return key <= pos and (window == 0 or key > pos - window or key < first)


@pytest.mark.parametrize("seed", range(12))
def test_every_row_and_part_once(seed):
    r = random.Random(seed)
    for _ in range(15):
        n_seq = r.randint(1, 30)
        heads, kv, dim = r.choice(((64, 8, 64), (28, 4, 80), (8, 1, 128), (16, 16, 64), (40, 1, 64)))
        group = heads // kv
        lengths = [r.choice((r.randint(1, 200), r.randint(1, 20000))) for _ in range(n_seq)]
        counts = [r.choice((1, r.randint(1, min(n, 700)))) for n in lengths]
        window = r.choice((0, 0, r.randint(1, 3000)))
        (size, tokens, at_items, items, at_joins, joins, part_rows, nbytes, at_weights, w_items, w_joins, w_parts), out = plan(
            counts, lengths, heads, kv, dim, window, r.randint(0, 50) if window else 0)
        starts = np.concatenate(([0], np.cumsum(counts)))
        assert tokens == sum(counts) and out[:n_seq + 1].tolist() == starts.tolist()
        assert at_items >= n_seq + 1 and at_joins == at_items + 8 * items and at_weights == at_joins + 8 * joins
        assert size == at_weights + 4 * w_items
        assert (out[size:] == -7).all() and nbytes == part_rows * kv * (4 * dim + 16)
        rows, parts, splits_of = set(), {}, {}
        for s, begin, count, row0, n, split, splits, part in out[at_items:at_joins].reshape(-1, 8).tolist():
            assert begin == starts[s] and count == counts[s] and 0 < n <= 128 and 0 <= split < splits
            for x in range(n):
                assert row0 + x < counts[s] * group
                key = (s, row0 + x, split)
                assert key not in rows
                rows.add(key)
                splits_of[s, row0 + x] = splits
                if splits > 1:
                    at = part + split * n + x
                    assert 0 <= at < part_rows and at not in parts
                    parts[at] = key
        assert set(splits_of) == {(s, x) for s in range(n_seq) for x in range(counts[s] * group)}
        assert len(rows) == sum(splits_of.values()) and len(parts) == part_rows
        seen = set()
        for s, begin, count, row0, n, splits, part, stride in out[at_joins:at_weights].reshape(-1, 8).tolist():
            assert begin == starts[s] and count == counts[s] and 0 < n <= 16
            for x in range(n):
                for p in range(splits):
                    assert parts[part + x + p * stride] == (s, row0 + x, p)
                    seen.add(part + x + p * stride)
        assert seen == set(parts)
        of, places = {}, []
        for i, (s, part, n, offset) in enumerate(out[at_weights:size].reshape(-1, 4).tolist()):
            assert 0 <= part < n <= -(-counts[s] * group // 256) and (i < w_joins) == (n > 1 and part == 0)
            of.setdefault(s, []).append(part)
            places += [offset + part] if n > 1 else []
            assert n == 1 or out[at_weights:size].reshape(-1, 4)[i, 3] == offset
        assert {s: sorted(x) for s, x in of.items()} == {s: list(range(len(x))) for s, x in of.items()} and len(of) == n_seq
        assert sorted(places) == list(range(w_parts))


def span(keys_a_tile, p_lo, p_hi, window, first):
    """The kernels' list of tiles for rows at positions p_lo..p_hi, and the key that stands for each key of a tile."""
    low = max(0, p_lo - window + 1) // 16 * 16 if window else 0
    head = (min(first, max(p_hi, 0)) + 15) // 16 * 16
    if head >= low:
        head = low = 0
    head_tiles = -(-head // keys_a_tile)
    low_tile = max(low // keys_a_tile, head_tiles)
    tiles = 0 if p_hi < 0 else head_tiles + p_hi // keys_a_tile + 1 - low_tile
    bases = [(j if j < head_tiles else j - head_tiles + low_tile) * keys_a_tile for j in range(tiles)]

    def at(base, key):
        gap = head - 1 if base < head_tiles * keys_a_tile else low
        return min(key, p_hi) if key >= low else key if key < head else gap

    return bases, at


def test_the_tiles_hold_what_is_seen_and_nothing_else():
    """A model of the tiles' arithmetic: every seen key once, only pages that some row sees, and rows of one load
    instruction (8 keys) in one page."""
    r = random.Random(3)
    for i in range(4000):
        kt, group, n = r.choice((32, 64)), r.choice((1, 2, 4, 7, 8)), r.randint(1, 400)
        count = r.randint(1, min(n + 3, 60))
        window = r.choice((0, r.randint(1, 450)))
        first = r.randint(0, 100) if window else 0
        base, row0 = n - count, r.choice(range(0, count * group, 128))
        p_lo, p_hi = base + row0 // group, base + (min(row0 + 128, count * group) - 1) // group
        bases, at = span(kt, p_lo, p_hi, window, first)
        held = []
        for b in bases:
            for k in range(b, b + kt, 8):
                piece = [at(b, k + e) for e in range(8)]
                assert len({x // 16 for x in piece}) == 1 and 0 <= min(piece) and max(piece) < n
                of = piece[0] // 16 * 16
                assert any(sees(p, x, window, first) for p in range(p_lo, p_hi + 1) for x in range(of, of + 16))
            held += [k for k in range(b, b + kt) if at(b, k) == k]
        assert len(held) == len(set(held))
        assert {k for p in range(max(p_lo, 0), p_hi + 1) for k in range(p + 1) if sees(p, k, window, first)} <= set(held)


def test_asking_for_the_size_and_too_little_room():
    sizes, _ = plan([3, 1], [5000, 9000], capacity=0)
    again, out = plan([3, 1], [5000, 9000], capacity=int(sizes[0]) - 1)
    assert again == sizes and (out == -7).all()
    exact, out = plan([3, 1], [5000, 9000], capacity=int(sizes[0]))
    assert exact == sizes and out[:3].tolist() == [0, 3, 4]


@pytest.mark.parametrize("kw", [
    dict(counts=[0], lengths=[5]), dict(counts=[-1], lengths=[5]), dict(counts=[6], lengths=[5]), dict(counts=[1], lengths=[1 << 29]),
    dict(counts=[1], lengths=[5], window=-1), dict(counts=[1], lengths=[5], first=2), dict(counts=[1], lengths=[5], window=3, first=-1),
    dict(counts=[1], lengths=[5], heads=7, kv=2), dict(counts=[1], lengths=[5], dim=60), dict(counts=[1], lengths=[5], dim=136),
    dict(counts=[1], lengths=[5], heads=0), dict(counts=[1 << 28], lengths=[1 << 28])])
def test_plan_refusals(kw):
    with pytest.raises(nat.KlcError) as e:
        plan(**kw)
    assert e.value.status in (nat.KLC_ERR_ARGUMENT, nat.KLC_ERR_SHAPE) and "klc_attn_plan" in e.value.message


def test_plan_python_refusals():
    for args, error in ((([1, 2], [3]), ValueError), (([], []), ValueError), (([[1]], [[2]]), ValueError), (([1.0], [2]), TypeError),
                        (([1], ["a"]), TypeError), (([0], [1]), ValueError), (([2], [1]), ValueError), (([1], [1 << 29]), ValueError)):
        with pytest.raises(error):
            ops.attention_plan(*args, 8, 2, 64)
    for kw in (dict(window=0), dict(window=-1), dict(first=1), dict(window=4, first=-1)):
        with pytest.raises(ValueError):
            ops.attention_plan([1], [2], 8, 2, 64, **kw)
    with pytest.raises(TypeError):
        ops.attention_plan([1], [2], 8, 2, 64, window=1.5)
    with pytest.raises(ValueError, match="GPU"):
        ops.attention_plan([1], [2], 8, 2, 64, device="cpu")


FAKE = 0x1000  # never dereferenced: validation fails first


def refused(name, fields, layout, **change):
    values = {**fields, **change}
    with pytest.raises(nat.KlcError) as e:
        nat.call(name, struct.pack(layout, *values.values()), None)
    assert e.value.status in (nat.KLC_ERR_ARGUMENT, nat.KLC_ERR_SHAPE, nat.KLC_ERR_UNSUPPORTED) and name in e.value.message
    return e.value.message


CHUNK = dict(q=FAKE, k_pages=FAKE, v_pages=FAKE, tables=FAKE, lengths=FAKE, plan=FAKE, sinks=0, workspace=0, out=FAKE, lse=0, at_items=8,
             items=1, at_joins=16, joins=0, part_rows=0, n_heads=8, n_kv=2, head_dim=64, q_stride=512, n_pages=4, page_size=16,
             table_width=2, window=0, first=0, kv_dtype=1, workspace_bytes=0, scale=0.125)


@pytest.mark.parametrize("change", [
    dict(q=0), dict(k_pages=0), dict(v_pages=0), dict(tables=0), dict(lengths=0), dict(plan=0), dict(out=0), dict(q=FAKE + 8),
    dict(out=FAKE + 2), dict(lse=FAKE + 1), dict(items=0), dict(joins=-1), dict(part_rows=-1), dict(part_rows=5),
    dict(part_rows=5, workspace=FAKE, workspace_bytes=10), dict(n_heads=7), dict(n_kv=0), dict(head_dim=0), dict(head_dim=136),
    dict(head_dim=60), dict(q_stride=504), dict(q_stride=516), dict(n_pages=0), dict(n_pages=1 << 31), dict(page_size=8),
    dict(page_size=24), dict(page_size=8192), dict(table_width=-1), dict(table_width=1 << 26), dict(window=-1), dict(first=1),
    dict(window=5, first=-1), dict(kv_dtype=2), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=1e39),
    dict(n_kv=4096, n_heads=4096, head_dim=128, q_stride=1 << 20, page_size=4096)])
def test_chunk_refusals(change):
    refused("klc_attn_chunk", CHUNK, "=10Q16qd", **change)


WEIGHTS = dict(q=FAKE, lse=FAKE, k_pages=FAKE, tables=FAKE, lengths=FAKE, plan=FAKE, rows=FAKE, weights=FAKE, workspace=0, at_items=8, items=1,
               joins=0, parts=0, n_rows=1, capacity=64, n_heads=8, n_kv=2, head_dim=64, q_stride=512, n_pages=4, page_size=16, table_width=2,
               window=0, first=0, kv_dtype=1, workspace_bytes=0, scale=0.125)


@pytest.mark.parametrize("change", [
    dict(q=0), dict(lse=0), dict(k_pages=0), dict(tables=0), dict(lengths=0), dict(plan=0), dict(rows=0), dict(weights=0),
    dict(q=FAKE + 2), dict(weights=FAKE + 2), dict(items=0), dict(joins=-1), dict(joins=2), dict(parts=-1), dict(parts=2), dict(n_rows=0),
    dict(capacity=0), dict(n_heads=9), dict(head_dim=12), dict(q_stride=100), dict(page_size=17), dict(n_pages=-1), dict(window=-1),
    dict(first=3), dict(kv_dtype=5), dict(scale=0.0), dict(items=2, parts=2), dict(items=2, parts=2, workspace=FAKE, workspace_bytes=1023),
    dict(items=2, parts=2, workspace=FAKE + 4, workspace_bytes=1 << 40), dict(items=1 << 31), dict(items=1 << 23), dict(items=1 << 62), dict(n_heads=4096, n_kv=4096, head_dim=128, q_stride=1 << 20, page_size=4096)])
def test_key_weight_refusals(change):
    refused("klc_attn_key_weights", WEIGHTS, "=9Q17qd", **change)


EVICT = dict(pools=FAKE, weights=FAKE, tables=FAKE, lengths=FAKE, rows=FAKE, kept=FAKE, workspace=FAKE, n_layers=1, n_seq=1, n_rows=1,
             capacity=64, n_kv=2, head_dim=64, n_pages=4, page_size=16, table_width=2, keep=10, recent=2, first=1, workspace_bytes=1 << 20)


@pytest.mark.parametrize("change", [
    dict(pools=0), dict(weights=0), dict(tables=0), dict(lengths=0), dict(rows=0), dict(kept=0), dict(workspace=0), dict(pools=FAKE + 8),
    dict(weights=FAKE + 1), dict(n_layers=0), dict(n_seq=0), dict(n_rows=0), dict(capacity=0), dict(n_kv=0), dict(head_dim=20),
    dict(n_pages=0), dict(page_size=48), dict(table_width=0), dict(keep=0), dict(keep=-1), dict(recent=-1), dict(first=-1),
    dict(recent=9, first=2), dict(workspace_bytes=79), dict(keep=1 << 29, workspace_bytes=1 << 50)])
def test_evict_refusals(change):
    refused("klc_kv_evict", EVICT, "=7Q13q", **change)


NORM = dict(q=FAKE, k=FAKE, v=FAKE, cos=FAKE, sin=FAKE, positions=FAKE, slots=FAKE, q_out=FAKE, k_out=0, k_pages=FAKE, v_pages=FAKE, tokens=1,
            n_positions=10, n_slots=16, n_heads=8, n_kv=2, head_dim=64, q_stride=512, k_stride=128, v_stride=128, kv_dtype=1, q_norm=FAKE,
            k_norm=FAKE, eps=1e-6)


@pytest.mark.parametrize("change", [dict(q=0), dict(q_out=0), dict(positions=0), dict(q_norm=FAKE + 2), dict(k_norm=FAKE + 8), dict(eps=-1.0),
                                    dict(eps=float("nan")), dict(eps=float("inf")), dict(head_dim=12), dict(kv_dtype=2), dict(tokens=0)])
def test_norm_append_refusals(change):
    refused("klc_kv_norm_append", NORM, "=11Q10q2Qd", **change)


def test_null_arguments():
    for name in ("klc_attn_chunk", "klc_attn_key_weights", "klc_kv_evict", "klc_kv_norm_append"):
        with pytest.raises(nat.KlcError, match="null pointer"):
            nat.call(name, None, None)


def test_one_long_sequence_among_many_is_cut():
    """Whatever the others are: the longest keys set the time of a plan that leaves them whole."""
    lengths = [200 + 6 * i for i in range(127)] + [32000]
    sizes, out = plan([1] * 128, lengths)
    splits = {int(x[0]): int(x[6]) for x in out[sizes[2]:sizes[4]].reshape(-1, 8)}
    assert splits[127] >= 8 and max(splits[s] for s in range(127)) == 1
