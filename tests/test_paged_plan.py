"""The paged attention's division of work, restated without a GPU: the decode
kernel's shares cover every block of keys of every item once and leave their
states where the merge reads them; the prompt kernel's slots belong to one
block of one sequence each; starts and lengths of any values reach no row, page
or state out of range."""

import re
from pathlib import Path

import numpy as np
import pytest

LIMIT = 1 << 30
SOURCES = Path(__file__).resolve().parents[1] / "pdum_dsl_amd" / "csrc"
ITEM, LEAST = map(int, re.search(r"ITEM = (\d+), LEAST = (\d+);", (SOURCES / "paged_attn.hip").read_text()).groups())


def _seq(starts, lengths, i, rows):
    r0, r1 = (min(max(int(s), 0), rows) for s in starts[i : i + 2])
    return r0, max(0, r1 - r0), min(max(int(lengths[i]), 0), LIMIT)


def _plan(starts, lengths, i, rows, group, reach, window, sinks, per_block, keys=32):
    """row0, n, first position, row blocks, first-token blocks, window's first block, blocks."""
    r0, n, ln = _seq(starts, lengths, i, rows)
    pos0 = ln - n
    end = min(ln, reach)
    eb = -(-end // keys)
    wb = min(max(pos0 - window + 1, 0) // keys, eb)
    sb = min(-(-min(sinks, end) // keys), wb)
    return r0, n, pos0, -(-n * group // per_block), sb, wb, max(sb + eb - wb, 1)


def _shares(plans, heads, grid, item_cost=ITEM, least=LEAST):
    """What each workgroup sweeps: (workgroup, sequence, item, first block, end block, its record or None, cut's last)."""
    cost = [p[3] * (p[6] + item_cost) * heads for p in plans]
    total = sum(cost)
    per = -(-total // grid)
    per = -(-per // 4) * 4 if per > least else least
    ends = np.cumsum([0] + cost)
    out = []
    for w in range(grid):
        at, left = per * w, min(total - per * w, per)
        if left <= 0:
            continue
        seq = int(np.searchsorted(ends, at, side="right")) - 1
        units = plans[seq][6] + item_cost
        item, unit = divmod(int(at - ends[seq]), units)
        while left > 0:
            units = plans[seq][6] + item_cost - unit
            take = min(units, left)
            kb, end = max(unit - item_cost, 0), max(unit + take - item_cost, 0)
            if end == 0:
                break
            whole = end - kb == plans[seq][6]
            last = (at + units - 1) // per if kb == 0 and not whole else None
            out.append((w, seq, item, kb, end, None if whole else 2 * w + (kb == 0), last))
            left, at, unit = left - take, at + take, unit + take
            if take == units and left > 0:
                unit, item = 0, item + 1
                if item == plans[seq][3] * heads:
                    item, seq = 0, seq + 1
                    while plans[seq][1] == 0:
                        seq += 1
    return out, per


CASES = [(lengths, new, group, heads, window, sinks, grid)
         for lengths, new in (([1], [1]), ([1000], [1]), ([7, 0, 33, 5000, 1], [1, 0, 1, 1, 1]), ([40] * 300, [1] * 300),
                              ([100000, 32, 32, 64], [3, 1, 2, 5]), ([9, 8], [9, 8]), (list(range(1, 700)), [1] * 699))
         for group, heads in ((1, 1), (4, 8), (20, 2)) for window, sinks in ((LIMIT, 0), (50, 4)) for grid in (512, 768)]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_every_block_is_swept_once_and_every_state_found(case):
    lengths, new, group, heads, window, sinks, grid = CASES[case]
    starts = np.concatenate([[0], np.cumsum(new)])
    rows = int(starts[-1])
    plans = [_plan(starts, lengths, i, rows, group, 1 << 17, window, sinks, 16) for i in range(len(lengths))]
    got, per = _shares(plans, heads, grid)
    swept, records = {}, {}
    for w, seq, item, kb, end, rec, last in got:
        assert 0 <= kb < end <= plans[seq][6]
        assert swept.get((seq, item), 0) == kb  # in order, without a gap
        swept[seq, item] = end
        if rec is not None:
            assert rec < 2 * grid and rec not in records
            records[rec] = (seq, item)
    for i, p in enumerate(plans):
        for item in range(p[3] * heads):
            assert swept[i, item] == p[6]
    owners = {(s, it): (w, last) for w, s, it, kb, end, rec, last in got if last is not None}
    for key in {k for k in records.values()}:  # a cut item: its owner's second record, then first ones up to `last`
        w, last = owners[key]
        mine = sorted(r for r, k in records.items() if k == key)
        assert mine == sorted([2 * w + 1] + [2 * x for x in range(w + 1, last + 1)])
        assert last < grid


def _slot(starts, seqs, rows, group, slot):
    base = [min(max(int(starts[i]), 0), rows) * group // 128 + i for i in range(seqs + 1)]
    n = sum(b <= slot for b in base) - 1
    return n, (slot - base[n] if n >= 0 else 0)


@pytest.mark.parametrize("new,pad", [([1], 0), ([500, 0, 0, 3, 128, 129], 0), ([1] * 50, 7), ([0, 0, 4096], 100), ([31, 33, 64], 1)])
@pytest.mark.parametrize("group", [1, 4, 7, 20])
def test_every_block_has_one_slot(new, pad, group):
    starts = np.concatenate([[0], np.cumsum(new)])
    rows = int(starts[-1]) + pad
    seqs = len(new)
    seen = {}
    for slot in range(rows * group // 128 + seqs + 1):
        seq, rb = _slot(starts, seqs, rows, group, slot)
        n = 0 if seq < 0 else (new + [pad])[seq]
        if seq >= 0 and 0 <= rb < -(-n * group // 128):
            assert (seq, rb) not in seen
            seen[seq, rb] = slot
    for i, n in enumerate(new + [pad]):
        for rb in range(-(-n * group // 128)):
            assert (i, rb) in seen


def test_any_starts_and_lengths_stay_in_range():
    rng = np.random.default_rng(0)
    lo, hi = -(2**31), 2**31 - 1
    for _ in range(400):
        seqs, rows, group = int(rng.integers(1, 9)), int(rng.integers(1, 300)), int(rng.integers(1, 9))
        pick = lambda n: np.where(rng.random(n) < 0.5, rng.integers(-5, 400, n), rng.integers(lo, hi, n))  # noqa: E731
        starts, lengths = pick(seqs + 1), pick(seqs)
        window = int(rng.choice([1, 7, LIMIT]))
        width, page = int(rng.integers(0, 5)), 16
        for i in range(seqs):
            for per_block in (16, 128):
                r0, n, pos0, nb, sb, wb, blocks = _plan(starts, lengths, i, rows, group, width * page, window, 3, per_block)
                assert 0 <= r0 and r0 + n <= rows and nb * per_block < 2**31
                assert 0 <= sb <= wb and 1 <= blocks <= LIMIT // 32
                for v in (0, blocks - 1):  # the table's entries that the first and last block read
                    key = (v if v < sb else v - sb + wb) * 32
                    for h in (0, 16):
                        e = min((key + h) // page, max(width, 1) - 1)
                        assert 0 <= e < max(width, 1)
                assert lo <= pos0 - window + 1 and pos0 + n + 31 <= hi
        for slot in range(rows * group // 128 + seqs + 1):
            seq, rb = _slot(starts, seqs, rows, group, slot)
            assert -1 <= seq <= seqs
            if 0 <= seq < seqs:
                r0, n, *_ = _plan(starts, lengths, seq, rows, group, 64, LIMIT, 0, 128)
                if 0 <= rb < -(-n * group // 128):
                    assert r0 + (rb * 128) // group < rows


def _head_slot(bid, heads, nslots):
    """The prompt kernel's workgroup -> (head, slot), None where it has none; and the grid."""
    shares = 1
    while heads * shares % 8:
        shares *= 2
    units, unit_slots, run_of = heads * shares // 8, -(-nslots // shares), 3
    grid = 8 * units * unit_slots
    r, per_run = bid >> 3, run_of * unit_slots
    first, in_run = r // per_run * run_of, r % per_run
    n = min(units - first, run_of)
    if n <= 0:
        return None, grid
    unit = (bid & 7) * units + first + in_run % n
    j = in_run // n
    if (j | 3) < unit_slots and j & 4:
        j ^= 3
    j = j * shares + unit % shares
    return ((unit // shares, nslots - 1 - j) if j < nslots else None), grid


@pytest.mark.parametrize("heads", [1, 2, 3, 5, 8, 12, 16, 32, 40])
@pytest.mark.parametrize("nslots", [1, 2, 7, 67, 131])
def test_every_head_and_slot_has_one_workgroup(heads, nslots):
    grid = _head_slot(0, heads, nslots)[1]
    got = [x for x in (_head_slot(b, heads, nslots)[0] for b in range(grid)) if x is not None]
    assert sorted(got) == [(h, s) for h in range(heads) for s in range(nslots)]


def test_prompt_tiles_are_laid_out_as_the_forward_kernels():
    """The swizzles of the prompt kernel's tiles are the forward kernel's, whose reads other tests hold to no bank conflicts."""
    def body(name, file):
        return re.search(r"int %s\(int row\) \{\s*return (.*?);\s*\}" % name, (SOURCES / file).read_text(), re.S).group(1)

    for paged, dense in (("key_swizzle", "swz16_k"), ("value_swizzle", "swz16_v")):
        assert body(paged, "paged_attn.hip") == body(dense, "flash_fwd.hip")
