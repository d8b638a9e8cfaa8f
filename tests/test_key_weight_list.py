"""The host's list of the key weights' workgroups: a model of what the kernel makes of it, for the lengths that it was made
for and others; its size; and its refusals (no GPU)."""

from __future__ import annotations

import random
import struct

import numpy as np
import pytest

from klcquant_amd import _native as nat

KEYS, TILE = 256, 32  # of a block, of rows


def made(counts, lengths, heads=64, kv=8, dim=64, window=0, first=0):
    """(plan, its sizes, list, its sizes)"""
    counts, lengths = np.array(counts, np.int32), np.array(lengths, np.int32)
    sizes, of_list = np.zeros(12, np.int64), np.zeros(4, np.int64)
    args = (len(counts), heads, kv)
    plan_args = (counts.ctypes.data, lengths.ctypes.data, *args, dim, window, first)
    nat.call("klc_attn_plan", *plan_args, None, 0, sizes.ctypes.data)
    plan = np.zeros(sizes[0], np.int32)
    nat.call("klc_attn_plan", *plan_args, plan.ctypes.data, plan.size, sizes.ctypes.data)
    list_args = (plan.ctypes.data, sizes.ctypes.data, lengths.ctypes.data, *args, window, first)
    nat.call("klc_attn_weight_list", *list_args, None, 0, of_list.ctypes.data)
    asked, out = of_list.tolist(), np.full(of_list[0] + 8, -7, np.int32)
    nat.call("klc_attn_weight_list", *list_args, out.ctypes.data, int(of_list[0]) - 1, of_list.ctypes.data)
    assert of_list.tolist() == asked and (out == -7).all()
    nat.call("klc_attn_weight_list", *list_args, out.ctypes.data, int(of_list[0]), of_list.ctypes.data)
    assert of_list.tolist() == asked and (out[asked[0]:] == -7).all() and asked[0] == 8 * asked[1]
    return plan, sizes.tolist(), out[:asked[0]], asked


def up(a, b):
    return -(-a // b)


class Blocks:
    """The blocks of a sequence's keys, and the rows that see one."""

    def __init__(self, n, count, g, window, first):
        self.n, self.count, self.g, self.window, self.base = n, count, g, window, n - count
        self.heads = up(min(first, n), KEYS) if window else 0
        self.low = max(self.heads, max(0, self.base - window + 1) // KEYS if window else 0)
        self.end = up(n, KEYS)

    def rows(self, block):
        last = self.count - 1
        if self.window and block >= self.heads:
            last = min(last, min(self.n, (block + 1) * KEYS) - 1 + self.window - 1 - self.base)
        return max(0, block * KEYS - self.base) * self.g, (last + 1) * self.g

    def parts(self, head, most, least):
        tokens = self.count if head or not self.window else min(self.count, self.window + KEYS - 1)
        return min(most, up(up(tokens * self.g, TILE), least))


def check(counts, planned, lengths, heads, kv, window, first):
    """Every row that sees a block of keys once, over the blocks of `lengths`, from a list made for `planned`."""
    plan, sizes, of, (_, items, joins, scratch) = made(counts, planned, heads, kv, 64, window, first)
    g, least = heads // kv, int(of[7])
    records = {(s, part): most for s, part, most, _ in plan[sizes[8]:sizes[0]].reshape(-1, 4).tolist()}
    done, places = {}, {}
    for i, (s, part, parts, place, at, begin, count, tiles) in enumerate(of.reshape(-1, 8).tolist()):
        assert tiles == least >= 8 and (s, part) in records and begin == sum(counts[:s]) and count == counts[s]
        head, last, index = bool(place & 1), bool(place & 2), place >> 2
        keys = Blocks(lengths[s], counts[s], g, window, first)
        assert parts == keys.parts(head, records[s, part], least) > part and (i < joins) == (parts > 1 and part == 0)
        begin, end = (0, keys.heads) if head else (keys.low, keys.end)
        listed = block = begin + index
        while block < end:
            row, stop = keys.rows(block)
            per = max(up(up(stop - row, TILE), parts), least) * TILE if parts > 1 else max(stop - row, 0)
            if block != listed:
                per, part = max(stop - row, 0), 0
            if row + part * per < stop:
                for r in range(row + part * per, min(row + (part + 1) * per, stop)):
                    assert (s, block, r) not in done
                    done[s, block, r] = True
                if parts > 1 and block == listed:
                    assert 0 <= at < scratch and at not in places
                    places[at] = (s, block, part)
            if i < joins and block == listed:  # the second launch's sums, from here on
                held = up(max(stop - row, 0), max(per, 1))
                joined = [(at + p, (s, block, p)) for p in range(held)]
                assert held <= parts
                done.setdefault("joins", []).extend(joined)
            if not last or part > 0:
                break
            block += 1
    joined = done.pop("joins", [])
    assert dict(joined) == places and len(joined) == len(places)
    want = set()
    for s, n in enumerate(lengths):
        for t in range(counts[s]):
            p = n - counts[s] + t
            if p < 0:
                continue
            blocks = set(range((max(0, p - window + 1) if window else 0) // KEYS, p // KEYS + 1))
            blocks |= set(range(up(min(first, p + 1), KEYS))) if window else set()
            want |= {(s, b, t * g + h) for b in blocks for h in range(g)}
    # rows beside them that see nothing of a block (other ones of its keys' tokens) do no harm: they are masked
    assert want <= set(done)
    return items, scratch


@pytest.mark.parametrize("seed", range(8))
def test_every_row_of_every_block_once(seed):
    r = random.Random(seed)
    for _ in range(12):
        n_seq = r.randint(1, 6)
        heads, kv = r.choice(((64, 8), (28, 4), (8, 1), (16, 16), (40, 1)))
        planned = [r.choice((r.randint(1, 300), r.randint(1, 4000))) for _ in range(n_seq)]
        counts = [r.choice((1, r.randint(1, min(n, 900)))) for n in planned]
        window = r.choice((0, 0, r.randint(1, 600), 128))
        first = r.choice((0, 1, 4, r.randint(1, 700))) if window else 0
        check(counts, planned, planned, heads, kv, window, first)
        check(counts, planned, [n + r.choice((0, 1, 63, 300, 2000)) for n in planned], heads, kv, window, first)
        check(counts, planned, [r.randint(0, n) for n in planned], heads, kv, window, first)


def test_one_part_of_all_rows_of_steps():
    items, scratch = check([1] * 64, [1000 + 16 * i for i in range(64)], [1000 + 16 * i for i in range(64)], 64, 8, 0, 0)
    assert items == sum(up(1000 + 16 * i, KEYS) for i in range(64)) and scratch == 0


@pytest.mark.parametrize("counts,lengths,window,first", [
    # suffixes beside one step over very many keys
    ([100] * 64 + [1], [600] * 64 + [131072], 0, 0), ([1000] * 64 + [1], [4000] * 64 + [131072], 128, 4),
    ([1000] * 256 + [1], [4000] * 256 + [131072], 128, 4), ([1] * 4095 + [1], [200] * 4095 + [131072], 0, 0),
    ([1] * 127 + [1], [200 + 6 * i for i in range(127)] + [32000], 0, 0),
    # chunks behind many keys, a window and first tokens
    ([2000] * 30, [26000] * 30, 128, 4), ([1000] * 12, [25000] * 12, 128, 4), ([4000] * 64, [4000] * 64, 128, 4), ([1], [131072], 128, 4),
    # long chunks of one sequence, whose parts fill the chip
    ([6000], [8000], 0, 0), ([4096], [4096], 0, 0), ([6000], [8000], 128, 4), ([32000], [32000], 0, 0)])
def test_the_work_goes_by_what_each_sequence_sees(counts, lengths, window, first):
    """Not by the longest sequence of the batch, nor by first tokens for all keys.  A block of at most T tiles of rows has
    at most T / least + 1 parts.  The least is an eighth of a CU's tiles of the estimated work, which is no less than half
    of the blocks' T together (the new tokens' own blocks have half of the rows on average), so that all blocks have at
    most one part each and twice eight a CU more."""
    heads, kv = 64, 8
    _, _, _, (_, items, _, parts) = made(counts, lengths, heads, kv, window=window, first=first)
    blocks = 0
    for n, count in zip(lengths, counts):
        keys = Blocks(n, count, heads // kv, window, first)
        blocks += keys.heads + max(1, keys.end - keys.low)
    assert blocks <= items <= blocks + 2 * 8 * 256 // kv and parts <= items
    assert 2048 * parts * kv <= 2048 * kv * (blocks + 512)  # bytes of the second launch's sums: 8.4 MB and a block's 16 KB each


def test_refusals():
    plan, sizes, of, _ = made([3, 1], [5000, 9000])
    sizes, lengths, out = np.array(sizes), np.array([5000, 9000], np.int32), np.zeros(4, np.int64)

    def refused(**change):
        a = {**dict(plan=plan.ctypes.data, sizes=sizes.ctypes.data, lengths=lengths.ctypes.data, n_seq=2, heads=64, kv=8, window=0, first=0,
                    list=None, capacity=0, out=out.ctypes.data), **change}
        with pytest.raises(nat.KlcError, match="klc_attn_weight_list") as e:
            nat.call("klc_attn_weight_list", *a.values())
        assert e.value.status == nat.KLC_ERR_ARGUMENT

    for change in (dict(plan=None), dict(sizes=None), dict(lengths=None), dict(out=None), dict(capacity=5), dict(n_seq=0), dict(n_seq=1),
                   dict(heads=7), dict(kv=0), dict(heads=8192), dict(window=-1), dict(window=1 << 30), dict(first=1),
                   dict(window=4, first=-1), dict(window=4, first=1 << 29)):
        refused(**change)
    refused(heads=4096, kv=1, n_seq=1)  # not this plan's sequences
    keep, plan[0] = plan[0], 1
    refused()
    plan[0] = keep
    for bad in ([2, 9000], [5000, 0], [5000, -1], [1 << 29, 9000]):
        lengths[:] = bad
        refused()
    lengths[:] = [5000, 9000]
    for at, value in ((int(sizes[8]), 2), (int(sizes[8]), -1), (int(sizes[8]) + 1, 99), (int(sizes[8]) + 1, -1)):
        keep, plan[at] = plan[at], value
        refused()
        plan[at] = keep


def test_a_plans_records_are_no_list():
    """What an earlier interface passed, the records of the plan itself, is told from a list."""
    fake = 0x1000
    fields = [fake] * 8 + [0, 64, 2, 0, 0, 1, 64, 8, 2, 64, 512, 4, 16, 2, 0, 0, 1, 0, 0.125]
    with pytest.raises(nat.KlcError, match="not a list"):
        nat.call("klc_attn_key_weights", struct.pack("=9Q17qd", *fields), None)
