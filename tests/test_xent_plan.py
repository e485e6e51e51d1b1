"""The backward's plan of pdum_dsl_amd/csrc/xent.hip restated on the CPU: the
parts of dx (and of dw) that the last sums add are those that the products of
the first piece of the vocabulary write. The restatement is held to the
library's by the workspace's size, to the byte."""

import ctypes as C
import random

import pytest

BK, F32, BF16, F16 = 64, 0, 1, 2
TRY = (1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 14, 16, 20, 24, 28, 32, 40, 48, 56, 64)


def _ceil(a, b):
    return -(-a // b)


def _up(v, to):
    return _ceil(v, to) * to


def _slots():
    from pdum_dsl_amd import _lib

    return 2 * (_lib.lib().pdh_device_cus() or 256)


def _makespan(n1, d1, n2, d2, s):
    q, r = divmod(n1, s)
    early = q * d1
    late = early + (d1 if r else 0.0)
    if n2 == 0:
        return late if r else early
    i = 1
    while True:
        ends = [t for t in (early + i * d2, late + i * d2)
                if t >= late and (s - r) * int((t - early) / d2 + 1e-9) + r * max(0, int((t - late) / d2 + 1e-9)) >= n2]
        if ends:
            return min(ends)
        i += 1


def _plan(n, d, v, dtype, slots):
    """piece, the k columns of a slice of dw's and dx's products."""
    planes, dp = (3 if dtype == F32 else 1), _up(d, 8)
    most = (1 << 30) // (n * 2 * planes) // 256 * 256
    piece = min(_up(v, 256), 1 << 22, max(most, 256))
    bm, bn = (64, 256) if d <= 64 else (128, 256) if _ceil(d, 128) % 2 else (256, 128)
    mt = _ceil(d, bm)
    tw, tx = mt * _ceil(piece, bn), mt * _ceil(n, bn)
    terms = (6 if dtype == F32 else 1) * (0.6 if d <= 64 else 1.0)
    most_w = min(n // 512, (1 << 31) // (piece * dp * 4)) if tw < slots else 1
    most_x = min(piece // 256, (1 << 31) // (n * dp * 4))
    best, bw, bx = 1e300, 1, 1
    for w in TRY:
        if w > 1 and w > most_w:
            break
        dw = terms * _ceil(n, w * BK) + 5
        cost_w = 9e-7 * w * piece * dp + 2.5 if w > 1 else 0.0
        for x in TRY:
            if x > 1 and x > most_x:
                break
            dx = terms * _ceil(piece, x * BK) + 5
            t = cost_w + 9e-7 * x * n * dp + (_makespan(tx * x, dx, tw * w, dw, slots) if dx > dw
                                             else _makespan(tw * w, dw, tx * x, dx, slots))
            if t < best:
                best, bw, bx = t, w, x
    return piece, _up(_ceil(n, bw), BK), _up(_ceil(piece, bx), BK)


def _written(n, d, v, dtype, slots):
    """The workspace's bytes, with a part for each slice that the first piece's products launch."""
    piece, kw, kx = _plan(n, d, v, dtype, slots)
    planes, dp = (3 if dtype == F32 else 1), _up(d, 8)
    first = min(piece, v)
    parts_x, parts_w = _ceil(first, kx), _ceil(n, kw)
    assert (parts_x - 1) * kx < first and (parts_w - 1) * kw < n  # no slice without a column
    for v0 in range(0, v, piece):  # a later piece adds to parts that are there
        assert _ceil(min(piece, v - v0), kx) <= parts_x
    fit = dtype != F32 and d % 8 == 0  # w is read in place
    sizes = [] if fit else [v * dp * 2 * planes]
    sizes += [n * dp * 2 * planes, n * piece * 2 * planes, parts_x * n * dp * 4]
    if parts_w > 1:
        sizes.append(parts_w * piece * dp * 4)
    return sum(_up(s, 1024) for s in sizes + [4])


def _workspace(n, d, v, dtype):
    from pdum_dsl_amd import _lib

    p = C.c_void_p(256)
    return _lib.lib().pdh_linear_xent_workspace(p, p, n, d, v, d, d, dtype, 1)


@pytest.mark.parametrize("n,d,v,dtype", [
    (64, 1024, 16000, BF16), (8, 768, 16000, BF16), (1, 512, 16000, BF16), (300, 768, 8000, BF16), (300, 768, 8000, F16),
    (128, 512, 20000, F32), (600, 512, 30000, F32), (1030, 256, 30522, F32), (594, 1294, 2127, F32),
    (128, 1024, 30522, BF16), (1774, 128, 4462, BF16), (268, 448, 16923, BF16), (1326, 128, 2113, F32), (16, 768, 6657, BF16),
])
def test_every_part_that_is_summed_is_written(n, d, v, dtype):
    """Vocabularies whose last slice would lie wholly past their end if the slices were counted over whole tiles."""
    assert _workspace(n, d, v, dtype) == _written(n, d, v, dtype, _slots())


def test_every_part_that_is_summed_is_written_over_the_range():
    rng, slots = random.Random(1), _slots()
    log = lambda lo, hi: int(round(lo * (hi / lo) ** rng.random()))  # noqa: E731
    seen = 0
    while seen < 700:
        n, d, v, dtype = log(1, 20000), log(1, 5000), log(1, 300000), rng.choice((F32, BF16, F16))
        if rng.random() < 0.6:
            d = max(64, d // 64 * 64)
        if n * v > 1 << 32:
            continue
        seen += 1
        assert _workspace(n, d, v, dtype) == _written(n, d, v, dtype, slots), (n, d, v, dtype)


def test_several_pieces_write_every_part():
    for n, d, v, dtype in ((6000, 40, 200003, BF16), (3000, 200, 70001, F32), (5000, 500, 120001, F16), (120, 64, 5_000_000, BF16)):
        assert _plan(n, d, v, dtype, _slots())[0] < v
        assert _workspace(n, d, v, dtype) == _written(n, d, v, dtype, _slots())
