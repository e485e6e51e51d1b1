"""The paged-cache operators on the GPU against float64 closed forms
(oracle/paged.py): what an append stores and turns, what it leaves alone, and
attention over caches of 16 and 4 bits at the sizes, masks and layouts where
each can go wrong."""

import numpy as np
import pytest

from tests.paged_cases import batch, check_attention, half, op

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DT = {"bf16": torch.bfloat16, "f16": torch.float16}
MOST = {"bf16": 125, "f16": 13}


@pytest.fixture(scope="module")
def K():
    from pdum_dsl_amd import kernels

    return kernels


def _host(t):
    return t.detach().double().cpu().numpy()


def _ints(*arrays):
    return tuple(torch.as_tensor(a, dtype=torch.int32, device="cuda") for a in arrays)


def _pools(rng, K, dtype, bits, pages, heads, page_rows, d, std=1.0):
    """A cache of random contents and its values as float64 pools."""
    k, v = (torch.as_tensor(std * rng.standard_normal((pages, heads, page_rows, d))).to(DT[dtype]).cuda() for _ in range(2))
    if bits == 16:
        return K.PagedCache(k, v), _host(k), _host(v)
    parts, values = [], []
    for _ in range(2):
        codes = rng.integers(0, 16, (pages, heads, page_rows, d), dtype=np.uint8)
        scale = rng.integers(123, 128, (pages, heads, page_rows, d // 32), dtype=np.uint8)
        values.append(op.fp4_values(codes, scale))
        parts.append((torch.as_tensor(codes[..., 0::2] | (codes[..., 1::2] << 4)).cuda(), torch.as_tensor(scale).cuda()))
    (kc, ks), (vc, vs) = parts
    return K.PagedCache(kc, vc, ks, vs, DT[dtype]), *values


def _unpacked(codes):
    c = codes.cpu().numpy()
    return np.stack([c & 15, c >> 4], -1).reshape(c.shape[:-1] + (-1,))


# ---------------------------------------------------------------------- append

APPENDS = [
    # dtype, bits, lengths, new tokens, query heads, heads, features, page rows, rotated, interleaved, pad
    ("bf16", 16, [1], [1], 1, 1, 64, 16, 64, False, 0),
    ("f16", 16, [17, 5, 40, 40], [17, 0, 3, 1], 8, 2, 128, 16, 128, False, 0),
    ("bf16", 16, [100, 1], [70, 1], 12, 12, 64, 32, 32, True, 5),
    ("f16", 16, [64, 65], [1, 65], 5, 1, 128, 64, 16, False, 3),
    ("bf16", 16, [33], [33], 32, 8, 128, 16, 0, False, 0),
    ("bf16", 4, [1], [1], 4, 2, 128, 16, 128, False, 0),
    ("f16", 4, [50, 3, 18], [20, 3, 0], 3, 3, 64, 16, 64, True, 2),
    ("bf16", 4, [130], [129], 4, 4, 64, 128, 48, False, 1),
    ("f16", 4, [31, 32], [1, 32], 8, 1, 128, 32, 64, False, 0),
]


@pytest.mark.parametrize("case", APPENDS, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_append_matches_the_closed_form(K, case):
    dtype, bits, lengths, new, hq, hkv, d, pr, rotated, inter, pad = case
    rng = np.random.default_rng(len(str(case)))
    table, starts, lens, rows, pages = batch(rng, lengths, new, pr, pad=pad)
    cache, pk, pv = _pools(rng, K, dtype, bits, pages, hkv, pr, d)
    # one tensor holds q, k and v, as a projection leaves them
    qkv = torch.as_tensor(rng.standard_normal((rows, hq + 2 * hkv, d))).to(DT[dtype]).cuda()
    q, k, v = qkv[:, :hq], qkv[:, hq : hq + hkv], qkv[:, hq + hkv :]
    tab = op.rotary_table(max(lengths), rotated) if rotated else None
    before = [None if t is None else t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    bad = torch.zeros((), dtype=torch.int32, device="cuda")
    got = K.paged_append(k, v, cache, *_ints(table, starts, lens), q=q,
                         rotary=None if tab is None else torch.as_tensor(tab).cuda(), interleaved=inter, bad=bad)
    torch.cuda.synchronize()
    assert int(bad) == 0

    want_q = np.zeros((rows, hq, d))
    want = [b if b is None else b.clone() for b in before]
    hk, hv, hqv = (t.float().cpu().numpy() for t in (k, v, q))
    turn = lambda x, pos: op.rotate(x, tab[pos], inter) if rotated else x  # noqa: E731
    for r, i, pos in op.tokens(starts, lens, rows):
        page, at = op.place(table, i, pos, pr, pages)
        want_q[r] = torch.as_tensor(turn(hqv[r], pos)).to(DT[dtype]).double().numpy()
        for x, pool, scales in ((turn(hk[r], pos), 0, 2), (hv[r], 1, 3)):
            if bits == 16:
                want[pool][page, :, at] = torch.as_tensor(x).to(DT[dtype]).cuda()
            else:
                codes, sc = op.fp4(x, MOST[dtype])
                want[pool][page, :, at] = torch.as_tensor(codes[:, 0::2] | (codes[:, 1::2] << 4)).cuda()
                want[scales][page, :, at] = torch.as_tensor(sc).cuda()
    np.testing.assert_array_equal(_host(got), want_q)
    for t, w in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), want):
        assert t is None or torch.equal(t, w)  # the new tokens' places, and no other

    # and what the cache gives back is what it holds
    gk, gv = K.paged_rows(cache, *_ints(table, starts, lens), rows)
    values = [_host(cache.k), _host(cache.v)] if bits == 16 else [
        op.fp4_values(_unpacked(c), s.cpu().numpy()) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]
    for got_rows, pool in ((gk, values[0]), (gv, values[1])):
        w = np.zeros((rows, hkv, d))
        for r, i, pos in op.tokens(starts, lens, rows):
            page, at = op.place(table, i, pos, pr, pages)
            w[r] = pool[page, :, at]
        np.testing.assert_array_equal(_host(got_rows), w)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_four_bits_at_their_borders(K, dtype):
    """Ties, zeros of both signs, the largest and smallest numbers, infinities and NaN."""
    pr, d = 16, 64
    top = torch.finfo(DT[dtype]).max
    tiny = torch.finfo(DT[dtype]).smallest_normal
    rows = [
        [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, -7.0] * 2,  # ties
        [0.0, -0.0] * 16,
        [top, -top, top / 2, top / 4] * 8,
        [tiny, -tiny, tiny / 2, 0.0] * 8,
        [1.0] * 31 + [float("inf")],
        [2.0] * 31 + [float("nan")],
        [7.03125 if dtype == "bf16" else 7.0078125] + [0.5] * 31,  # the next number after 7: a larger scale
    ]
    x = torch.zeros((len(rows), 1, d))
    x[:, 0, :32] = torch.tensor(rows)
    x[:, 0, 32:] = 3.0  # the row's other group
    x = x.to(DT[dtype]).cuda()
    cache = K.paged_cache(2, 1, pr, d, DT[dtype], bits=4)
    t = _ints([[1]], [0, len(rows)], [len(rows)])
    K.paged_append(x, x, cache, *t)
    codes, scale = op.fp4(x.double().cpu().numpy(), MOST[dtype])
    for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        gc, gs = _unpacked(c)[1, 0, : len(rows)], s.cpu().numpy()[1, 0, : len(rows)]
        np.testing.assert_array_equal(gs, scale[:, 0])
        fine = np.repeat(gs != 255, 32, axis=-1)
        np.testing.assert_array_equal(gc[fine], codes[:, 0][fine])
    gk, _ = K.paged_rows(cache, *t, len(rows))
    got, want = _host(gk)[:, 0], op.fp4_values(codes, scale)[:, 0]
    want = torch.as_tensor(want).to(DT[dtype]).double().numpy()
    np.testing.assert_array_equal(got, want)
    assert np.isfinite(got[:4]).all() and np.isnan(got[4:6, :32]).all() and (got[4:6, 32:] == 3.0).all()
    finite = np.delete(got, [4, 5], 0)
    assert (np.abs(finite - np.delete(x.double().cpu().numpy()[:, 0], [4, 5], 0))[0] <= 1.0).all()  # half a step


def test_append_drops_tokens_without_a_place(K):
    """Pages outside the pool, tables that end, positions past the rotary table or below 0: counted, stored nowhere, and
    the other tokens are stored all the same."""
    pr, d, hkv, hq = 16, 64, 2, 4
    rng = np.random.default_rng(5)
    #        fine          a bad page        past the table  before 0   past the rotary table
    table = [[0, 1, 2], [3, 1 << 30, 4], [5, -7, -1], [6, 0, 0], [7, 8, 9]]
    lengths = [20, 40, 60, 2, 46]
    new = [2, 30, 3, 4, 4]
    starts = np.concatenate([[0], np.cumsum(new)])
    rows, pages, positions = int(starts[-1]), 10, 44
    cache = K.paged_cache(pages, hkv, pr, d)
    x = torch.as_tensor(rng.standard_normal((rows, hq + 2 * hkv, d))).to(torch.bfloat16).cuda()
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    tab = op.rotary_table(positions, d)
    got = K.paged_append(x[:, hq : hq + hkv], x[:, hq + hkv :], cache, *_ints(table, starts, lengths), q=x[:, :hq],
                         rotary=torch.as_tensor(tab).cuda(), bad=bad)
    want = np.zeros((pages, hkv, pr, d))
    want_q = np.zeros((rows, hq, d))
    dropped = 0
    for r, i, pos in op.tokens(starts, lengths, rows):
        w = op.place(np.array(table), i, pos, pr, pages)
        if w is None or pos >= positions:
            dropped += 1
            continue
        want[w[0], :, w[1]] = _host(x)[r, hq + hkv :]
        want_q[r] = torch.as_tensor(op.rotate(x[r, :hq].float().cpu().numpy(), tab[pos], False)).bfloat16().double().numpy()
    assert dropped and int(bad) == dropped
    np.testing.assert_array_equal(_host(cache.v), want)
    np.testing.assert_array_equal(_host(got), want_q)
    o, lse = K.paged_attention(got, cache, *_ints(table, starts, lengths))
    assert torch.isfinite(o.float()).all()
    k = _host(cache.k)
    w = op.attention(want_q, k, want, np.array(table), starts, lengths, scale=d**-0.5)
    check_attention(_host(o), _host(lse), w, "bf16", d, "bad pages")


def test_append_turns_q_in_place_and_leaves_other_rows(K):
    pr, d = 16, 128
    rng = np.random.default_rng(6)
    lengths, new, pad = [9, 30], [9, 2], 4
    table, starts, lens, rows, pages = batch(rng, lengths, new, pr, pad=pad)
    qkv = torch.as_tensor(rng.standard_normal((rows, 6, d))).half().cuda()
    tab = K.rotary_table(64, d)
    first = qkv.clone()
    outs = []
    for place in (None, "own", "q"):
        cache = K.paged_cache(pages, 1, pr, d, torch.float16)
        x = first.clone()
        out = None if place is None else (torch.full_like(x[:, :4], 7.0) if place == "own" else x[:, :4])
        got = K.paged_append(x[:, 4:5], x[:, 5:6], cache, *_ints(table, starts, lens), q=x[:, :4], rotary=tab, out=out)
        if out is not None:
            assert got is out
        outs.append(got.clone())
        assert torch.equal(x[:, 4:], first[:, 4:])
        tail = got[rows - pad :]
        want = torch.zeros_like(tail) if place is None else (torch.full_like(tail, 7.0) if place == "own" else first[rows - pad :, :4])
        assert torch.equal(tail, want)
    for o in outs[1:]:
        assert torch.equal(o[: rows - pad], outs[0][: rows - pad])


# ------------------------------------------------------------------- attention

ATTENDS = [
    # dtype, bits, lengths, new tokens, query heads, heads, features, page rows, window, sinks, pad
    # one token a sequence
    ("bf16", 16, [1], [1], 1, 1, 64, 16, None, 0, 0),
    ("bf16", 16, [1, 2, 15, 16, 17], [1] * 5, 8, 2, 128, 16, None, 0, 0),
    ("f16", 16, [31, 32, 33, 500], [1] * 4, 4, 4, 64, 32, None, 0, 1),
    ("bf16", 16, [3000, 7, 0, 1200], [1, 1, 0, 1], 32, 8, 128, 16, None, 0, 0),
    ("bf16", 16, [5000], [1], 12, 12, 64, 64, None, 0, 0),
    ("f16", 16, [2000, 999], [1, 1], 16, 1, 128, 16, None, 0, 0),
    ("bf16", 16, [700], [1], 40, 2, 64, 16, None, 0, 0),  # 20 query heads a head
    ("bf16", 16, [1500, 40], [1, 1], 8, 2, 128, 16, 100, 4, 0),
    ("f16", 16, [1500, 40, 3], [1, 1, 1], 8, 8, 64, 128, 1, 0, 0),
    ("bf16", 16, [1025, 90], [1, 1], 4, 1, 128, 32, 33, 50, 0),
    ("bf16", 4, [1, 33, 800], [1] * 3, 8, 2, 128, 16, None, 0, 0),
    ("f16", 4, [2500, 100], [1, 1], 4, 4, 64, 32, None, 0, 2),
    ("f16", 4, [2500, 100], [1, 1], 8, 1, 128, 64, 64, 3, 0),
    # a few tokens
    ("bf16", 16, [300, 4, 2000], [3, 4, 2], 8, 2, 128, 16, None, 0, 0),
    ("f16", 16, [300, 90], [5, 4], 6, 2, 64, 16, 20, 2, 3),
    ("bf16", 4, [600, 300], [4, 7], 4, 4, 128, 16, None, 0, 0),
    ("f16", 4, [333], [9], 5, 1, 64, 16, 40, 1, 0),
    # prompts and pieces of them, alone and beside single tokens
    ("bf16", 16, [33], [33], 2, 1, 64, 16, None, 0, 0),
    ("bf16", 16, [200, 31, 129], [200, 31, 129], 4, 2, 128, 16, None, 0, 0),
    ("f16", 16, [300, 700], [300, 100], 3, 3, 64, 32, None, 0, 7),
    ("bf16", 16, [1100], [600], 8, 2, 128, 64, 64, 4, 0),
    ("f16", 16, [500, 260], [500, 260], 7, 1, 128, 16, 150, 70, 0),
    ("bf16", 16, [900, 50, 400, 1], [300, 1, 1, 1], 8, 2, 64, 16, None, 0, 0),
    ("bf16", 4, [260, 300], [260, 41], 4, 2, 128, 16, None, 0, 0),
    ("f16", 4, [500], [333], 6, 3, 64, 128, 90, 5, 1),
    ("bf16", 4, [2048], [130], 16, 2, 64, 16, 1000, 0, 0),
]


def _attend(K, case, rng, poison=None, **kw):
    dtype, bits, lengths, new, hq, hkv, d, pr, window, sinks, pad = case
    table, starts, lens, rows, pages = batch(rng, lengths, new, pr, pad=pad)
    cache, pk, pv = _pools(rng, K, dtype, bits, pages, hkv, pr, d)
    if poison is not None:
        poison(cache, table, starts, lens)
    q = torch.as_tensor(rng.standard_normal((rows, hq, d))).to(DT[dtype]).cuda()
    got = K.paged_attention(q, cache, *_ints(table, starts, lens), window=window, sinks=sinks, **kw)
    every = max(1, max(new) // 60)
    want = op.attention(_host(q), pk, pv, table, starts, lens, scale=d**-0.5, window=window, sinks=sinks, every=every)
    return got, want, (q, cache, table, starts, lens)


@pytest.mark.parametrize("case", ATTENDS, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_attention_matches_the_closed_form(K, case):
    (o, lse), want, _ = _attend(K, case, np.random.default_rng(sum(case[2]) + case[4]))
    check_attention(_host(o), _host(lse), want, case[0], case[6], str(case))


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("case", [
    ("bf16", 16, [90, 33, 1], [1, 1, 1], 8, 2, 128, 16, None, 0, 0),
    ("f16", 16, [700, 40], [1, 1], 4, 4, 64, 16, 50, 3, 0),
    ("bf16", 4, [700, 40], [1, 1], 4, 2, 128, 16, 50, 3, 0),
    ("f16", 16, [300, 90], [4, 3], 4, 4, 64, 32, 40, 2, 0),
    ("bf16", 16, [300, 100], [200, 1], 4, 2, 128, 16, 45, 3, 0),
    ("f16", 4, [300, 100], [150, 100], 4, 2, 64, 16, 70, 0, 0),
], ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_what_no_row_sees_may_hold_anything(K, case, value):
    """Rows behind a sequence's end, pages of nobody, tokens between the first ones and every row's window."""
    dtype, bits, lengths, new, hq, hkv, d, pr, window, sinks, pad = case

    def poison(cache, table, starts, lens):
        pages = cache.k.shape[0]
        seen = np.zeros((pages, pr), dtype=bool)
        for i, n in enumerate(lens):
            first = n - (starts[i + 1] - starts[i])
            for s in range(n):
                if window is None or s > first - window or s < sinks:
                    seen[table[i, s // pr], s % pr] = True
        dead = torch.as_tensor(~seen, device="cuda")[:, None, :, None]
        for t in (cache.k, cache.v) if bits == 16 else (cache.k_scale, cache.v_scale):
            t.copy_(torch.where(dead, torch.tensor(value if bits == 16 else 255, device="cuda").to(t.dtype), t))

    (o, lse), want, _ = _attend(K, case, np.random.default_rng(3), poison)
    check_attention(_host(o), _host(lse), want, dtype, d, str(case))


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("new,hq,hkv", [([6, 1], 4, 4), ([2, 2], 8, 2), ([140, 33], 4, 2), ([70, 1], 3, 1)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (20, 1)])
def test_a_token_that_some_rows_see_spoils_those_alone(K, bits, new, hq, hkv, window, sinks):
    """A NaN in one token's value, an infinity in another's, a NaN in a key: every row that does not see them is what it
    is without them; every row that sees one is not finite."""
    pr, d = 16, 64
    rng = np.random.default_rng(8)
    lengths = [n + 50 for n in new]
    table, starts, lens, rows, pages = batch(rng, lengths, new, pr)
    cache, pk, pv = _pools(rng, K, "bf16", bits, pages, hkv, pr, d)
    q = torch.as_tensor(rng.standard_normal((rows, hq, d))).bfloat16().cuda()
    t = _ints(table, starts, lens)
    want = op.attention(_host(q), pk, pv, table, starts, lens, scale=d**-0.5, window=window, sinks=sinks)
    hurt = [lens[0] - 2, lens[0] - new[0] + 1, lens[0] - new[0] - 3]  # two of the first sequence's new tokens, an old one
    for s, (name, value) in zip(hurt, (("v", np.nan), ("v", np.inf), ("k", np.nan))):
        page, at = table[0, s // pr], s % pr
        if bits == 16:
            getattr(cache, name)[page, :, at, 5] = value
        else:
            getattr(cache, name + "_scale")[page, :, at, 0] = 255
    o, lse = K.paged_attention(q, cache, *t, window=window, sinks=sinks)
    o, lse = _host(o), _host(lse)
    spoiled = np.zeros(rows, dtype=bool)
    for r, i, pos in op.tokens(starts, lens, rows):
        if i == 0:
            spoiled[r] = any(s <= pos and (window is None or s > pos - window or s < sinks) for s in hurt)
    assert spoiled.any()
    keep = ~spoiled
    if keep.any():
        check_attention(o[keep], lse[keep], tuple(w[keep] for w in want), "bf16", d, "rows that do not see them")
    assert (~np.isfinite(o[spoiled])).any(-1).all()


def test_rows_that_see_nothing(K):
    """Sequences of no tokens, of fewer tokens than rows, and pages that are all outside the pool."""
    pr, d, hq, hkv = 16, 64, 4, 2
    rng = np.random.default_rng(9)
    for new in ([2, 1, 3], [40, 1, 90]):
        lengths = [0, 5, new[2] - 2]
        starts = np.concatenate([[0], np.cumsum(new)])
        rows = int(starts[-1])
        table = np.array([[0] * 8, [99] * 8, [1, 2, 3, 4, 5, 6, 7, 8]], dtype=np.int32)
        cache, pk, pv = _pools(rng, K, "bf16", 16, 9, hkv, pr, d)
        q = torch.as_tensor(rng.standard_normal((rows, hq, d))).bfloat16().cuda()
        o, lse = K.paged_attention(q, cache, *_ints(table, starts, lengths))
        want = op.attention(_host(q), pk, pv, table, starts, lengths, scale=d**-0.5)
        assert np.isneginf(want[1][: new[0] + new[1] + 2]).all()
        check_attention(_host(o), _host(lse), want, "bf16", d, f"new {new}")
        # no page at all in the table
        o, lse = K.paged_attention(q, cache, torch.empty((3, 0), dtype=torch.int32, device="cuda"), *_ints(starts, lengths))
        assert (o == 0).all() and torch.isneginf(lse).all()


def test_no_rows_and_no_sequences(K):
    cache = K.paged_cache(2, 2, 16, 64)
    q = torch.zeros((0, 4, 64), dtype=torch.bfloat16, device="cuda")
    o, lse = K.paged_attention(q, cache, *_ints([[0]], [0, 0], [7]))
    assert o.shape == q.shape and lse.shape == (0, 4)
    q = torch.ones((3, 4, 64), dtype=torch.bfloat16, device="cuda")
    empty = (torch.empty((0, 2), dtype=torch.int32, device="cuda"), *_ints([0], []))
    o, lse = K.paged_attention(q, cache, *empty)
    assert (o == 0).all() and torch.isneginf(lse).all()
    got = K.paged_append(q[:, :2], q[:, :2], cache, *empty, q=q)
    assert (got == 0).all() and (cache.k == 0).all()


@pytest.mark.parametrize("new", [[1, 1], [3, 60]])
def test_rows_of_no_sequence_stay_as_they_are_in_out(K, new):
    case = ("bf16", 16, [100, 120], new, 8, 2, 64, 16, None, 0, 37)
    (o, lse), want, (q, cache, table, starts, lens) = _attend(K, case, np.random.default_rng(2))
    rows = q.shape[0]
    assert (o[rows - 37 :] == 0).all() and torch.isneginf(lse[rows - 37 :]).all()
    # into a wider tensor's middle
    wide = torch.full((rows, 8, 192), 3.0, dtype=torch.bfloat16, device="cuda")
    out = wide[:, :, 64:128]
    got, _ = K.paged_attention(q, cache, *_ints(table, starts, lens), out=out, want_lse=False)
    assert got is out and torch.equal(out[: rows - 37], o[: rows - 37])
    assert (out[rows - 37 :] == 3.0).all() and (wide[:, :, :64] == 3.0).all() and (wide[:, :, 128:] == 3.0).all()


@pytest.mark.parametrize("new", [[1, 1, 1], [2, 100, 9]])
def test_pools_of_any_strides(K, new):
    """Heads behind rows, keys and values in one tensor, and rows of q by heads first: the same bits."""
    case = ("f16", 16, [200, 130, 17], new, 4, 2, 64, 16, None, 0, 0)
    (o, lse), want, (q, cache, table, starts, lens) = _attend(K, case, np.random.default_rng(4))
    both = torch.stack((cache.k, cache.v), 1).permute(0, 1, 3, 2, 4).contiguous()  # [pages, 2, page_rows, heads, features]
    other = K.PagedCache(both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2))
    q2 = q.transpose(0, 1).contiguous().transpose(0, 1)
    o2, lse2 = K.paged_attention(q2, other, *_ints(table, starts, lens))
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    check_attention(_host(o), _host(lse), want, "f16", 64, "strides")


def test_pages_past_32_bits(K):
    """Pages whose place in the pool passes 2^32 bytes."""
    pr, d, hkv, hq = 16, 64, 1, 4
    far = (1 << 32) // 2 // 4 + 8 * 1024  # elements from page to page: a pool spans 4 of these, over 4 GB
    rng = np.random.default_rng(10)
    k, v = (torch.zeros(far * 4 + pr * d, dtype=torch.bfloat16, device="cuda").as_strided((5, hkv, pr, d), (far, pr * d, d, 1))
            for _ in range(2))
    cache = K.PagedCache(k, v)
    lengths, new = [70, 33], [1, 33]
    table = np.array([[4, 0, 3, 1, 2], [2, 4, 1, 0, 3]], dtype=np.int32)[:, :5]
    for i in range(2):  # the second sequence's pages are the first's: one after the other
        starts, lens = np.array([0, lengths[i]]), np.array([lengths[i]])
        x = torch.as_tensor(rng.standard_normal((lengths[i], hkv, d))).bfloat16().cuda()
        K.paged_append(x, x, cache, *_ints(table[i : i + 1], starts, lens))
        q = torch.as_tensor(rng.standard_normal((new[i], hq, d))).bfloat16().cuda()
        o, lse = K.paged_attention(q, cache, *_ints(table[i : i + 1], [0, new[i]], lens))
        hk, hv = np.zeros((5, hkv, pr, d)), np.zeros((5, hkv, pr, d))
        for r in range(lengths[i]):
            p, at = op.place(table[i : i + 1], 0, r, pr, 5)
            hk[p, :, at] = hv[p, :, at] = _host(x[r])
        want = op.attention(_host(q), hk, hv, table[i : i + 1], [0, new[i]], lens, scale=d**-0.5)
        check_attention(_host(o), _host(lse), want, "bf16", d, f"far pages {i}")


# ---------------------------------------------- as a program uses them


@pytest.mark.parametrize("bits", [16, 4])
def test_prompts_then_steps_equal_the_whole(K, bits):
    """Prompts go in by pieces, then tokens one at a time; what each step's rows see, and the cache in the end, is what one
    call over everything gives."""
    pr, d, hq, hkv = 16, 64, 8, 2
    rng = np.random.default_rng(12)
    lengths = [75, 40]
    table, _, _, _, pages = batch(rng, lengths, [1, 1], pr)
    x = [torch.as_tensor(rng.standard_normal((n, hq + 2 * hkv, d))).bfloat16().cuda() for n in lengths]
    tab = K.rotary_table(128, d)

    def step(cache, spans):
        part = torch.cat([x[i][a:b] for i, (a, b) in enumerate(spans)])
        starts = np.concatenate([[0], np.cumsum([b - a for a, b in spans])])
        t = _ints(table, starts, [b for _, b in spans])
        q = K.paged_append(part[:, hq : hq + hkv], part[:, hq + hkv :], cache, *t, q=part[:, :hq], rotary=tab)
        o, lse = K.paged_attention(q, cache, *t, window=30, sinks=2)
        return [(o[starts[i] : starts[i + 1]], lse[starts[i] : starts[i + 1]]) for i in range(2)]

    whole = K.paged_cache(pages, hkv, pr, d, bits=bits)
    all_o = step(whole, [(0, n) for n in lengths])
    cache = K.paged_cache(pages, hkv, pr, d, bits=bits)
    got = [[], []]
    for spans in [[(0, 50), (0, 20)], [(50, 70), (20, 36)]] + [[(70 + j, 71 + j), (min(36 + j, 40), min(37 + j, 40))] for j in range(5)]:
        for i, part in enumerate(step(cache, spans)):
            got[i].append(part)
    for a, b in ((cache.k, whole.k), (cache.v, whole.v), (cache.k_scale, whole.k_scale)):
        assert a is None or torch.equal(a, b)
    # each is within its bound of the exact row: twice a rounding of a factor and of the result apart
    t = _ints(table, [0, 75, 115], lengths)
    kk, vv = (_host(r) for r in K.paged_rows(whole, *t, 115))
    top = max(np.abs(vv).max(), 1.0)
    for i in range(2):
        o = torch.cat([p[0] for p in got[i]])
        lse = torch.cat([p[1] for p in got[i]])
        assert np.abs(_host(o) - _host(all_o[i][0])).max() <= 4 * half("bf16") * top
        assert np.abs(_host(lse) - _host(all_o[i][1])).max() <= 1e-4


def test_two_streams_and_repeats(K):
    """Two calls at once on streams of their own, each with its own workspace: the bits of calls one after the other."""
    cases = [("bf16", 16, [3000, 500], [1, 1], 8, 2, 128, 16, None, 0, 0), ("bf16", 4, [900], [300], 8, 2, 128, 16, 200, 4, 0)]
    want, args = [], []
    for n, c in enumerate(cases):
        (o, lse), _, (q, cache, table, starts, lens) = _attend(K, c, np.random.default_rng(n))
        args.append((q, cache, *_ints(table, starts, lens)))
        want.append((o, lse))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(10):
        for n, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[n].append(K.paged_attention(*args[n], window=cases[n][8], sinks=cases[n][9]))
    torch.cuda.synchronize()
    for n in range(2):
        for o, lse in got[n]:
            assert torch.equal(o, want[n][0]) and torch.equal(lse, want[n][1])


@pytest.mark.parametrize("bits", [16, 4])
def test_a_captured_step_follows_its_inputs(K, bits):
    """One decode step as a graph: replays read the table, starts and lengths of the moment, and give the eager bits."""
    pr, d, hq, hkv = 16, 128, 8, 2
    rng = np.random.default_rng(13)
    table, starts, lens, rows, pages = batch(rng, [200, 40, 9], [1, 1, 1], pr, width=16)
    cache, *_ = _pools(rng, K, "bf16", bits, pages, hkv, pr, d)
    x = torch.as_tensor(rng.standard_normal((rows, hq + 2 * hkv, d))).bfloat16().cuda()
    tab = K.rotary_table(256, d)
    t = _ints(table, starts, lens)

    def step(c):
        q = K.paged_append(x[:, hq : hq + hkv], x[:, hq + hkv :], c, *t, q=x[:, :hq], rotary=tab)
        return K.paged_attention(q, c, *t, sinks=2, window=64)

    step(cache)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = step(cache)
    for n in range(4):
        x.copy_(torch.as_tensor(rng.standard_normal(tuple(x.shape))).bfloat16())
        t[2].copy_(torch.tensor([200 - 3 * n, 40 - n, 9 + n], dtype=torch.int32))
        other = K.PagedCache(*(None if p is None else p.clone() for p in (cache.k, cache.v, cache.k_scale, cache.v_scale)),
                             torch.bfloat16)
        eo, el = step(other)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, eo) and torch.equal(lse, el), n
        assert torch.equal(cache.k, other.k) and torch.equal(cache.v, other.v)
