"""The tile loop of pdum_dsl_amd/csrc/xent.hip restated on the CPU: its direct
loads fill each LDS tile once and stay inside it and inside the operand (the
rest reads as zero), its fragment reads give the matrix instruction the rows
and k columns that the epilogues assume, and no read meets a bank twice."""

import itertools

import pytest

from tests.test_lds_layout import _ways

BK, OOB = 64, 1 << 31


def _swz(R, kc, row):
    if kc:
        return (row & 7) ^ ((row >> 3) & 1)
    return 4 * (row & 3) if R >= 128 else 4 * ((row >> 1) & 1)


def _fill(R, kc, rows, k, k0, k1, pitch):
    """LDS byte -> operand element (row, k) or None (zero) for one k tile of rows 0 .. R - 1."""
    last = k1 - k0 < BK
    nr, nk = min(rows, R), (k1 - k0 if last else BK)
    ext = (nr - 1) * pitch + ((nk * 2 + 15) & ~15) if kc else (nk - 1) * pitch + ((nr * 2 + 15) & ~15)
    ktail = (k1 - k0) % BK
    lds = {}
    slots = BK * 2 // 16 if kc else R // 8
    nrows = 64 // slots
    for w, i in itertools.product(range(4), range(R * BK * 2 // 1024 // 4)):
        blk = 4 * i + w
        for lane in range(64):
            row = lane // slots
            chunk = (lane % slots) ^ _swz(R, kc, nrows * w + row)
            voff = row * pitch + 16 * chunk
            if kc and last and not 8 * chunk < ktail:
                voff = OOB
            soff = nrows * blk * pitch
            for b in range(0, 16, 2):
                at = voff + soff + b
                assert blk * 1024 + lane * 16 + b not in lds
                inside = at < ext
                if inside:
                    r, c = divmod(at, pitch)
                    lds[blk * 1024 + lane * 16 + b] = (r, k0 + c // 2) if kc else (c // 2, k0 + r)
                else:
                    lds[blk * 1024 + lane * 16 + b] = None
    assert len(lds) * 2 == R * BK * 2 and max(lds) < R * BK * 2
    return lds


def _perm(r):
    return 16 * ((r >> 2) & 1) + 4 * (r >> 3) + (r & 3)


def _reads(R, T, kc, perm, wq, t, ks):
    """The lanes' LDS addresses (b128, or the first tr read's) of a fragment: block 0's 32 t rows on, or step 0's 16 ks k rows on."""
    out = []
    for lane in range(64):
        if kc:
            r, g = lane & 31, lane >> 5
            row = 32 * wq * T + (_perm(r) if perm else r)
            out.append(row * BK * 2 + (((2 * ks + g) ^ _swz(R, kc, row)) << 4) + 32 * t * BK * 2)
        else:
            G, i4 = lane >> 4, (lane >> 2) & 3
            q = 4 * (G & 1) + (lane & 3)
            kr = 8 * (G >> 1) + i4
            col = 32 * (wq * T + t) + (16 * (q & 1) + 4 * (q >> 1) if perm else 4 * q)
            out.append(kr * R * 2 + (((col >> 3) ^ _swz(R, kc, kr)) << 4) + ((col >> 2) & 1) * 8 + 16 * ks * R * 2)
    return out


def _fragment(lds, R, T, kc, perm, wq, t, ks):
    """The (row, k) of each lane's eight values."""
    addr = _reads(R, T, kc, perm, wq, t, ks)
    if kc:
        return [[lds[a + 2 * j] for j in range(8)] for a in addr]
    out = []
    for lane in range(64):
        G, i = lane >> 4, lane & 15
        vals = []
        for half in (0, 4 * R * 2):
            for k in range(4):  # chunk addressed by lane 4 k + i / 4 of the group, element i % 4
                vals.append(lds[addr[16 * G + 4 * k + i // 4] + half + 2 * (i % 4)])
        out.append(vals)
    return out


@pytest.mark.parametrize("R,T", [(256, 4), (256, 2), (128, 2), (128, 4), (64, 1), (64, 2)])
@pytest.mark.parametrize("kc", [True, False])
@pytest.mark.parametrize("perm", [True, False])
def test_fragments_hold_the_rows_and_columns_the_epilogues_assume(R, T, kc, perm):
    waves = R // (32 * T)
    if waves < 1:
        pytest.skip("no wave of this shape")
    for rows, k0, k1 in ((R, 0, 128), (R - 57, 64, 128), (3, 64, 81), (R, 0, 8), (R + 40, 64, 121)):
        # a k-contiguous operand's rows and a rows-contiguous one's k rows are whole 16-byte chunks of zeros past the end
        pitch = (max(k1, 128) if kc else ((rows + 7) & ~7)) * 2
        lds = _fill(R, kc, rows, 128, k0, k1, pitch)
        for wq, t, ks in itertools.product(range(waves), range(T), range(BK // 16)):
            got = _fragment(lds, R, T, kc, perm, wq, t, ks)
            for lane in range(64):
                r, g = lane & 31, lane >> 5
                row = 32 * (wq * T + t) + (_perm(r) if perm else r)
                for j in range(8):
                    k = k0 + 16 * ks + 8 * g + j
                    v = got[lane][j]
                    if row < rows and k < k1:
                        assert v == (row, k)
                    elif row < rows and v is not None:  # past k1: zero, or the zeros that end the operand's own chunk
                        assert kc and v == (row, k) and k < (k1 + 7) & ~7  # (rows past the last feed no output)


@pytest.mark.parametrize("R,T", [(256, 4), (256, 2), (128, 2), (128, 4), (64, 1), (64, 2)])
@pytest.mark.parametrize("perm", [True, False])
def test_no_read_meets_a_bank_twice(R, T, perm):
    for kc, width in ((True, 16), (False, 8)):
        for wq, t, ks in itertools.product(range(R // (32 * T)), range(T), range(BK // 16)):
            assert _ways(_reads(R, T, kc, perm, wq, t, ks), width) == 1


def test_an_accumulator_lane_holds_sixteen_consecutive_rows():
    """v_mfma_f32_32x32x16 gives register i of lane l row 8 (i / 4) + 4 (l / 32) + i % 4; the dealt rows make
    that row 16 (l / 32) + i of the tile."""
    for g, i in itertools.product(range(2), range(16)):
        assert _perm(8 * (i >> 2) + 4 * g + (i & 3)) == 16 * g + i


def test_the_pairs_of_terms_grow():
    pa = [(0x0118 >> (2 * i)) & 3 for i in range(6)]
    pb = [(0x0052 >> (2 * i)) & 3 for i in range(6)]
    assert list(zip(pa, pb)) == [(0, 2), (2, 0), (1, 1), (0, 1), (1, 0), (0, 0)]


def _run_ids(first, second):
    c1, c2 = (first + 7) // 8, (second + 7) // 8
    for bid in range((c1 + c2) * 8):
        xcd, pos = bid & 7, bid >> 3
        in2 = pos >= c1
        i = xcd * c2 + pos - c1 if in2 else xcd * c1 + pos
        if (pos - c1 < c2 and i < second) if in2 else i < first:
            yield in2, i


def _tile(tm, tn, i):
    s, i = divmod(i, tm * tn)
    group = min(8, tn)
    g, rem = divmod(i, group * tm)
    gn = min(tn - g * group, group)
    return s, rem // gn, g * group + rem % gn


def test_every_tile_is_taken_once():
    for first, second in itertools.product((0, 1, 7, 8, 9, 513), (0, 1, 30, 64)):
        ids = list(_run_ids(first, second))
        assert sorted(ids) == [(False, i) for i in range(first)] + [(True, i) for i in range(second)]
    for tm, tn, sl in itertools.product((1, 3, 20, 197), (1, 2, 7, 8, 9, 33), (1, 5)):
        assert {_tile(tm, tn, i) for i in range(tm * tn * sl)} == set(
            itertools.product(range(sl), range(tm), range(tn)))


@pytest.mark.parametrize("es,tm", [(2, 4), (4, 4), (2, 2)])
def test_stored_rows_leave_lds_as_they_came(es, tm):
    """put_rows: each lane's sixteen-column runs come back as whole rows, from a part of LDS no larger than its own,
    without bank conflicts."""
    pitch, ch = tm * 32 * es, tm * 32 * es // 16
    at_once, sw = (16 if es == 4 else 32), (ch - 1 if ch < 16 else 15)
    assert 4 * at_once * pitch <= 32768
    seen = set()
    for r0 in range(0, 32, at_once):
        lds = {}
        for i, q in itertools.product(range(tm), range(es)):
            offs = {}
            for lane in range(64):
                mine = lane & 31
                if not r0 <= mine < r0 + at_once:
                    continue
                c = (i * 32 + 16 * (lane >> 5)) * es // 16 + q
                at = (mine - r0) * pitch + ((c ^ (mine & sw)) << 4)
                assert at not in lds and at + 16 <= at_once * pitch
                lds[at] = (mine, 32 * i + 16 * (lane >> 5) + 16 // es * q)  # row, first column
                offs[lane] = at
            if len(offs) == 64 and ch >= 16:
                assert _ways([offs[lane] for lane in range(64)], 16) == 1
        for it in range(at_once * ch // 64):
            offs = []
            for lane in range(64):
                r, c = divmod(it * 64 + lane, ch)
                row = r0 + r
                offs.append(r * pitch + ((c ^ (row & sw)) << 4))
                assert lds[offs[-1]] == (row, c * 16 // es)
                seen.add((row, c))
            assert ch < 16 or _ways(offs, 16) == 1
    assert len(seen) == 32 * ch
