"""What the paged-cache calls refuse to write: the host's arithmetic on strided rows, compiled from its header and held
against every byte of small arrays, and the refusals of the C entry points (each fires before any HIP call)."""

import ctypes as C
import random
import subprocess
from pathlib import Path

import pytest

from tests.test_paged_ops import FAKE, _four_bits, _structs

CSRC = Path(__file__).resolve().parents[1] / "pdum_dsl_amd" / "csrc"

MAIN = """
#include "spans.h"
#include <cstdio>
using pdh::Spans;
static bool read(Spans& s) {
  long long at, width, n[4], st[4];
  if (scanf("%lld %lld", &at, &width) != 2) return false;
  for (int i = 0; i < 4; ++i) scanf("%lld %lld", &n[i], &st[i]);
  s = Spans(reinterpret_cast<const void*>(at), width, {{n[0], st[0]}, {n[1], st[1]}, {n[2], st[2]}, {n[3], st[3]}});
  return true;
}
int main() {
  Spans a(nullptr, 1, {});
  while (read(a)) printf("%d\\n", a.apart());
}
"""

PAIRS = MAIN.split("int main()")[0] + """
int main() {
  Spans a(nullptr, 1, {}), b = a;
  while (read(a) && read(b)) printf("%d\\n", a.apart_from(b) ? b.apart_from(a) : b.apart_from(a) ? 2 : 0);
}
"""


def _run(tmp_path, main, arrays):
    (tmp_path / "spans.cpp").write_text(main)
    exe = tmp_path / "spans"
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", str(CSRC), str(tmp_path / "spans.cpp"), "-o", str(exe)], check=True)
    text = "\n".join(" ".join(map(str, (at, width, *[x for axis in axes for x in axis]))) for at, width, axes in arrays)
    out = subprocess.run([str(exe)], input=text, check=True, capture_output=True, text=True).stdout
    return [bool(int(line)) for line in out.split()]


def _rows(at, axes):
    starts = [at]
    for n, step in axes:
        starts = [s + i * step for s in starts for i in range(n)]
    return starts


def _draw(rng):
    """Axes of a few entries, half of the time each stepping over the ones before it, by little or much."""
    width, axes = rng.choice([4, 8, 64]), []
    extent = width
    for _ in range(4):
        n = rng.choice([1, 1, 2, 3, 5])
        step = extent * rng.choice([1, 1, 2, 3]) + rng.choice([0, 0, 4]) if rng.random() < 0.8 else rng.randrange(0, 300)
        axes.append((n, step))
        extent = max(extent, (n - 1) * step + extent)
    rng.shuffle(axes)
    return rng.randrange(0, 400), width, axes


def test_no_array_that_overlaps_is_taken_for_apart(tmp_path):
    rng = random.Random(1)
    arrays = [_draw(rng) for _ in range(3000)]
    got = _run(tmp_path, MAIN, arrays)
    right = 0
    for (at, width, axes), apart in zip(arrays, got):
        starts = sorted(_rows(at, axes))
        truth = all(b - a >= width for a, b in zip(starts, starts[1:]))
        assert truth or not apart, (at, width, axes)
        ordered, extent = sorted((s, n) for n, s in axes if n > 1), width
        nested = True
        for s, n in ordered:
            nested &= s >= extent
            extent += (n - 1) * s
        assert apart == nested, (at, width, axes)  # nothing that nests is refused
        right += truth and apart
    assert right > 1000


def test_no_two_arrays_that_overlap_are_taken_for_apart(tmp_path):
    """Drawn pairs, half of them cut from one tensor as a projection's q, k and v are, those of which are always told apart."""
    rng = random.Random(2)
    arrays, views = [], []
    for _ in range(4000):
        if rng.random() < 0.5:
            arrays += [_draw(rng), _draw(rng)]
            views.append(False)
            continue
        rows, d, gap = rng.choice([1, 2, 7]), rng.choice([4, 16]), rng.choice([0, 0, 4])
        parts = [rng.choice([1, 2, 5]) for _ in range(3)]
        heads = sum(parts)
        if rng.random() < 0.5:  # rows of heads, or heads of rows
            st, sh = heads * d + gap, d
        else:
            st, sh = d, rows * d + gap
        at = rng.randrange(0, 4) * 64
        both = rng.sample(range(3), 2)
        arrays += [(at + sum(parts[:i]) * sh, d, [(rows, st), (parts[i], sh), (1, 0), (1, 0)]) for i in both]
        views.append(True)
    got = _run(tmp_path, PAIRS, arrays)
    assert len(got) == len(views)
    seen = 0
    for a, b, apart, view in zip(arrays[::2], arrays[1::2], got, views):
        truth = all(x + a[1] <= y or y + b[1] <= x for x in _rows(a[0], a[2]) for y in _rows(b[0], b[2]))
        assert truth or not apart, (a, b)
        assert apart or not view, (a, b)
        seen += truth and apart and max(_rows(a[0], a[2])) > min(_rows(b[0], b[2]))
    assert seen > 1000


FAR = 1 << 24  # the values' pool, past the end of the keys'


def _append(cache, batch=None):
    from pdum_dsl_amd import _lib

    c, b = _structs(cache, batch)
    q = C.c_void_p(FAKE)
    rc = _lib.lib().pdh_paged_append(C.c_void_p(FAR), C.c_void_p(2 * FAR), q, q, 4, 256, 64, 256, 64, 256, 64, 256, 64, C.byref(c),
                                     C.byref(b), None, 0, 0, 0, 0, 1, None, None)
    return rc, _lib.last_error()


@pytest.mark.parametrize("cache", [
    dict(),  # keys and values in one tensor
    dict(v=FAKE + 64),  # values between keys
    dict(v=FAKE + 4 * 2048 * 2 - 128),  # the values' first row is the keys' last
    dict(v=FAR, sh=0),  # heads in one place
    dict(v=FAR, sp=0),  # pages in one place
    dict(v=FAR, sh=512),  # heads inside one another
    dict(v=FAR, sp=1024),  # a page starts in the one before
    dict(_four_bits(v=FAR), sp=1024, sh=512, ssp=64, ssh=32),  # scales of keys and values in one tensor
    dict(_four_bits(v=FAR), sp=1024, sh=512, v_scale=FAR // 2, ssp=32, ssh=32),  # scales' pages in one another
    dict(_four_bits(v=FAR), sp=1024, sh=512, v_scale=FAR // 2, ssp=64, ssh=0),
    dict(_four_bits(), sp=1024, sh=512, v_scale=FAR // 2, ssp=64, ssh=32),  # codes of keys and values in one tensor
])
def test_an_append_to_rows_that_overlap_is_refused(cache):
    from pdum_dsl_amd import _lib

    rc, text = _append(cache)
    assert rc == _lib.PDH_EINVAL and "overlap" in text, (rc, text)
    assert _append(cache, dict(rows=0))[0] == _lib.PDH_OK  # nothing to store


@pytest.mark.parametrize("out,st,sh", [
    (FAKE + 512, 256, 64),  # q, a row on
    (FAKE + 128, 256, 64),  # a head on
    (FAKE, 512, 64),  # q's place, with other strides
    (FAKE, 256, 128),
    (FAR, 256, 64),  # k
    (2 * FAR + 64, 256, 64),  # v
    (FAR - 256, 256, 64),  # its end lies in k
    (4 * FAR, 64, 64), (4 * FAR, 0, 64),  # rows in one another
])
def test_results_that_overlap_inputs_are_refused(out, st, sh):
    from pdum_dsl_amd import _lib

    lib, q = _lib.lib(), C.c_void_p(FAKE)
    c, b = _structs(dict(k=8 * FAR, v=16 * FAR))
    rc = lib.pdh_paged_append(C.c_void_p(FAR), C.c_void_p(2 * FAR), q, C.c_void_p(out), 4, 256, 64, 256, 64, 256, 64, st, sh,
                              C.byref(c), C.byref(b), None, 0, 0, 0, 0, 1, None, None)
    assert rc == _lib.PDH_EINVAL and "overlap" in _lib.last_error(), (rc, _lib.last_error())
    if FAR - 256 <= out < 4 * FAR:
        return
    rc = lib.pdh_paged_attention(q, C.c_void_p(out), None, 4, 256, 64, st, sh, C.byref(c), C.byref(b), 5, 0, 1.0, 1,
                                 C.c_void_p(32 * FAR), 1 << 40, None)
    assert rc == _lib.PDH_EINVAL and "overlap" in _lib.last_error(), (rc, _lib.last_error())


@pytest.mark.parametrize("v,st,sh", [(FAR, 128, 64), (FAR + 64, 128, 64), (FAR - 1024, 128, 64), (2 * FAR, 64, 64), (2 * FAR, 128, 0)])
def test_read_back_rows_that_overlap_are_refused(v, st, sh):
    from pdum_dsl_amd import _lib

    c, b = _structs()
    rc = _lib.lib().pdh_paged_rows(C.c_void_p(FAR), C.c_void_p(v), 128, 64, st, sh, C.byref(c), C.byref(b), 1, None)
    assert rc == _lib.PDH_EINVAL and "overlap" in _lib.last_error(), (rc, _lib.last_error())


@pytest.mark.parametrize("bits,at", [(16, FAR), (16, 2 * FAR), (16, FAR + 6144), (16, 2 * FAR - 1024), (4, FAR), (4, 2 * FAR + 2048),
                                     (4, 3 * FAR), (4, 4 * FAR + 64)])
def test_results_in_the_cache_are_refused(bits, at):
    from pdum_dsl_amd import _lib

    lib, far = _lib.lib(), C.c_void_p(32 * FAR)
    kind = dict() if bits == 16 else dict(bits=4, sp=1024, sh=512, sr=32, ssp=64, ssh=32, ssr=2, k_scale=3 * FAR, v_scale=4 * FAR)
    c, b = _structs(dict(k=FAR, v=2 * FAR, **kind))
    out, more, other = C.c_void_p(at), C.c_void_p(33 * FAR), C.c_void_p(34 * FAR)
    for call in (
        lambda: lib.pdh_paged_append(more, more, far, out, 4, 256, 64, 256, 64, 256, 64, 256, 64, C.byref(c), C.byref(b), None, 0, 0,
                                     0, 0, 1, None, None),
        lambda: lib.pdh_paged_rows(out, far, 128, 64, 128, 64, C.byref(c), C.byref(b), 1, None),
        lambda: lib.pdh_paged_rows(far, out, 128, 64, 128, 64, C.byref(c), C.byref(b), 1, None),
        lambda: lib.pdh_paged_attention(far, out, None, 4, 256, 64, 256, 64, C.byref(c), C.byref(b), 5, 0, 1.0, 1, other, 1 << 40,
                                        None),
        lambda: lib.pdh_paged_attention(far, out, None, 32, 32 * 64, 64, 32 * 64, 64, C.byref(c), C.byref(b), 5, 0, 1.0, 1, other,
                                        1 << 40, None),
    ):
        assert call() == _lib.PDH_EINVAL and "overlap" in _lib.last_error(), _lib.last_error()


@pytest.mark.parametrize("width,heads,group", [(1 << 18, 64, 2), (1 << 18, 1, 4), (1 << 12, 64, 2)])
def test_work_that_could_pass_a_64_bit_sum_is_refused(width, heads, group):
    """The decode kernel sums up all sequences' work before it looks for its own. Starts that do not ascend can give every
    sequence all rows, and the sum then passes 2^63: no share of it would be found."""
    from pdum_dsl_amd import _lib

    rows, seqs, page = (1 << 24) // group, 1 << 20, 4096
    work = seqs * (rows * group // 16) * heads * (width * page // 32)  # of 2^20 sequences of all rows
    assert work > 1 << 63
    c, b = _structs(dict(heads=heads, sp=heads * page * 64, sh=page * 64, page_rows=page, v=FAR),
                    dict(seqs=seqs, rows=rows - 1, width=width, ld_table=0))
    hq, q = heads * group, C.c_void_p(2 * FAR)
    rc = _lib.lib().pdh_paged_attention(q, q, None, hq, hq * 64, 64, hq * 64, 64, C.byref(c), C.byref(b), 1 << 40, 0, 1.0, 1, q,
                                        1 << 40, None)
    assert rc == _lib.PDH_EINVAL and "work" in _lib.last_error(), (rc, _lib.last_error())
