"""The paged-cache operators on the GPU where a table, starts or lengths are not what a call means: pages that are missing,
rows that no sequence owns, sequences that go on behind the call's rows, lengths past every table."""

import ctypes as C

import numpy as np
import pytest

from tests.paged_cases import batch, check_attention, op
from tests.test_gpu_paged import DT, _host, _ints, _pools

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def K():
    from pdum_dsl_amd import kernels

    return kernels


@pytest.mark.parametrize("dtype,bits", [("bf16", 16), ("f16", 16), ("bf16", 4), ("f16", 4)])
@pytest.mark.parametrize("missing", [-1, 1 << 20])
@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("window", [None, 70])
def test_a_missing_page_is_not_another_ones(K, dtype, bits, missing, half, window):
    """Single tokens beside a piece, each without one page of the last 32 keys that it should see whole: neither the first
    page of the pool nor the last, which hold infinities and NaN and are nobody's, stand in for it."""
    rng = np.random.default_rng(40)
    pr, d, hq, hkv = 16, 64, 8, 2
    lengths, new = [40, 104, 33, 96, 200, 150], [1, 1, 1, 1, 1, 100]
    table, starts, lens, rows, pages = batch(rng, lengths, new, pr)
    cache, pk, pv = _pools(rng, K, dtype, bits, pages, hkv, pr, d)
    used = set(table[table >= 0].tolist())
    free = sorted(set(range(pages)) - used)[:2]
    swap = {0: free[0], pages - 1: free[1]}  # pages 0 and the last are to be nobody's
    swap = {a: b for a, b in swap.items() if a in used}
    table = np.vectorize(lambda p: swap.get(p, p))(table).astype(np.int32)
    for i, n in enumerate(lengths):
        table[i, 2 * ((n >> 5) - 1) + half] = missing
    for page in (0, pages - 1):
        assert page not in table
        if bits == 16:
            cache.k[page], cache.v[page] = float("nan"), float("inf")
            cache.v[page, :, ::2] = float("nan")
        else:
            cache.k_scale[page] = cache.v_scale[page] = 255
    q = torch.as_tensor(rng.standard_normal((rows, hq, d))).to(DT[dtype]).cuda()
    o, lse = K.paged_attention(q, cache, *_ints(table, starts, lens), window=window, sinks=2)
    want = op.attention(_host(q), pk, pv, table, starts, lens, scale=d**-0.5, window=window, sinks=2)
    check_attention(_host(o), _host(lse), want, dtype, d, f"missing {missing}, half {half}")


@pytest.mark.parametrize("starts,lengths,rows", [
    ([0, 8], [8], 5), ([0, 3, 12], [20, 30], 7), ([0, 90], [150], 61), ([0, 1, 200, 300], [40, 210, 100], 130),
    ([0, 2**31 - 1], [2**31 - 1], 8), ([0, 2**31 - 1], [2**31 - 1], 40), ([0, 2**31 - 1], [30], 40),
])
@pytest.mark.parametrize("bits", [16, 4])
def test_sequences_that_go_on_behind_the_rows(K, starts, lengths, rows, bits):
    """A call of fewer rows than starts describes: the rows that are there have the positions that they would have."""
    rng = np.random.default_rng(41)
    pr, d, hq, hkv = 16, 64, 4, 2
    n, width = len(lengths), 14
    pages = n * width
    table = rng.permutation(pages).reshape(n, width).astype(np.int32)
    cache = K.paged_cache(pages, hkv, pr, d, bits=bits)
    whole, *_ = _pools(rng, K, "bf16", bits, pages, hkv, pr, d)
    for a, b in ((cache.k, whole.k), (cache.v, whole.v), (cache.k_scale, whole.k_scale), (cache.v_scale, whole.v_scale)):
        if a is not None:
            a.copy_(b)
    x = torch.as_tensor(rng.standard_normal((rows, hq + 2 * hkv, d))).bfloat16().cuda()
    tab = op.rotary_table(300, d)
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    t = _ints(table, starts, lengths)
    q = K.paged_append(x[:, hq : hq + hkv], x[:, hq + hkv :], cache, *t, q=x[:, :hq], rotary=torch.as_tensor(tab).cuda(), bad=bad)
    gk, gv = K.paged_rows(cache, *t, rows)
    want_q, dropped = np.zeros((rows, hq, d)), 0
    owned = np.zeros((pages, pr), dtype=bool)
    for r, i, pos in op.tokens(starts, lengths, rows):
        w = op.place(table, i, pos, pr, pages)
        if w is None:
            dropped += 1
            assert (gk[r] == 0).all() and (gv[r] == 0).all()
            continue
        owned[w] = True
        want_q[r] = torch.as_tensor(op.rotate(x[r, :hq].float().cpu().numpy(), tab[pos], False)).bfloat16().double().numpy()
        if bits == 16:
            assert torch.equal(cache.v[w[0], :, w[1]], x[r, hq + hkv :])
            assert torch.equal(gk[r], cache.k[w[0], :, w[1]]) and torch.equal(gv[r], x[r, hq + hkv :])
        else:
            codes, scale = op.fp4(_host(x[r, hq + hkv :]), 125)
            np.testing.assert_array_equal(_host(gv[r]), op.fp4_values(codes, scale))
    assert int(bad) == dropped
    np.testing.assert_array_equal(_host(q), want_q)
    for a, b in ((cache.k, whole.k), (cache.v, whole.v)):  # and nothing else is stored
        same = (a == b).all(-1).all(1).cpu().numpy()
        assert same[~owned].all()
    full = torch.arange(0, n * width * pr + 1, width * pr)
    kk, vv = (_host(y).reshape(pages, pr, hkv, d).transpose(0, 2, 1, 3) for y in K.paged_rows(
        cache, torch.arange(pages, dtype=torch.int32, device="cuda").view(n, width), *_ints(full, [width * pr] * n), pages * pr))
    for window, sinks in ((None, 0), (50, 3)):
        o, lse = K.paged_attention(q, cache, *t, window=window, sinks=sinks)
        want = op.attention(_host(q), kk, vv, table, starts, lengths, scale=d**-0.5, window=window, sinks=sinks)
        check_attention(_host(o), _host(lse), want, "bf16", d, f"{starts} {window}")


@pytest.mark.parametrize("rows", [5, 60])
def test_lengths_past_the_longest_table(K, rows):
    """A table of 2^30 tokens and lengths over that: tokens past it have no place, those before it keep theirs, and a window
    goes by the positions as they are."""
    rng = np.random.default_rng(42)
    pr, d, hq, hkv, reach = 4096, 64, 4, 2, 1 << 30
    table = torch.full((1, reach // pr), -1, dtype=torch.int32, device="cuda")
    table[0, -1] = 1
    cache, pk, pv = _pools(rng, K, "bf16", 16, 3, hkv, pr, d)
    x = torch.as_tensor(rng.standard_normal((rows, hq + 2 * hkv, d))).bfloat16().cuda()
    q, v = x[:, :hq], x[:, hq + hkv :]
    past = rows - 2
    for length, fits in ((reach + past, 2), (reach + 3 * rows, 0), (2**31 - 1, 0)):
        before = cache.v.clone()
        bad = torch.zeros(1, dtype=torch.int32, device="cuda")
        t = (table, *_ints([0, rows], [length]))
        K.paged_append(x[:, hq : hq + hkv], v, cache, *t, bad=bad)
        assert int(bad) == rows - fits
        want = before.clone()
        for r in range(fits):
            want[1, :, pr - fits + r] = v[r]
        assert torch.equal(cache.v, want)
        # the same by a table of the last page alone, with all positions 2^30 - 4096 earlier
        o, lse = K.paged_attention(q, cache, *t, window=500)
        near = [[1]], [0, rows], [min(length - reach + pr, 9000)]
        ref = op.attention(_host(q), _host(cache.k), _host(cache.v), np.array(near[0]), near[1], near[2], scale=d**-0.5, window=500)
        check_attention(_host(o), _host(lse), ref, "bf16", d, str(length))


@pytest.mark.parametrize("new", [[1, 2, 1], [2, 70, 130]])
@pytest.mark.parametrize("first", [1, 5, 70])
def test_rows_before_the_first_sequence_are_of_no_sequence(K, new, first):
    from pdum_dsl_amd import _lib

    rng = np.random.default_rng(43)
    pr, d, hq, hkv = 16, 64, 8, 2
    table, starts, lens, rows, pages = batch(rng, [90, 80, 200], new, pr, pad=2)
    starts, rows = starts + first, rows + first
    cache, pk, pv = _pools(rng, K, "bf16", 16, pages, hkv, pr, d)
    q = torch.as_tensor(rng.standard_normal((rows, hq, d))).bfloat16().cuda()
    t = _ints(table, starts, lens)
    want = op.attention(_host(q), pk, pv, table, starts, lens, scale=d**-0.5)
    o, lse = K.paged_attention(q, cache, *t)
    check_attention(_host(o), _host(lse), want, "bf16", d, "starts that begin later")
    b = _lib.PagedBatch(t[0].data_ptr(), t[1].data_ptr(), t[2].data_ptr(), 3, rows, table.shape[1], table.shape[1])
    need = _lib.lib().pdh_paged_attention_workspace(C.byref(cache.c), C.byref(b), hq, 1 << 40, 0)
    ws = torch.full((need // 4 + 4,), float("nan"), device="cuda")
    owned = torch.zeros(rows, dtype=torch.bool, device="cuda")
    owned[first:-2] = True
    for rest in (1, 0):
        o2, l2 = torch.full_like(q, 9.0), torch.full((rows, hq), 9.0, device="cuda")
        _lib.call("pdh_paged_attention", q.data_ptr(), o2.data_ptr(), l2.data_ptr(), hq, hq * d, d, hq * d, d, C.byref(cache.c),
                  C.byref(b), 1 << 40, 0, d**-0.5, rest, ws.data_ptr(), need, K._stream())
        assert torch.equal(o2[owned], o[owned]) and torch.equal(l2[owned], lse[owned])
        if rest:
            assert (o2[~owned] == 0).all() and torch.isneginf(l2[~owned]).all()
        else:
            assert (o2[~owned] == 9.0).all() and (l2[~owned] == 9.0).all()


def _layouts(pages, hkv, pr, d):
    """Keys' and values' views of one tensor, and of two, in the orders that programs hold them in; d: bytes or features."""
    def make(*shape):
        return torch.zeros(shape, dtype=torch.uint8, device="cuda")

    both = make(pages, 2, hkv, pr, d)
    yield both[:, 0], both[:, 1]
    yield both[:, 1], both[:, 0]  # the values before the keys
    both = make(2, pages, hkv, pr, d)
    yield both[0], both[1]
    both = make(pages, pr, hkv, 2 * d)
    yield both[..., :d].transpose(1, 2), both[..., d:].transpose(1, 2)
    both = make(pages, pr, 2 * hkv, d).transpose(1, 2)
    yield both[:, :hkv], both[:, hkv:]
    yield both[:, ::2], both[:, 1::2]
    both = make(2 * pages, hkv, pr, d)
    yield both[::2], both[1::2]
    yield make(pages, hkv, pr, d), make(pages, hkv, pr, d)
    both = make(hkv, pages + 3, pr, d).transpose(0, 1)
    yield both[:pages], make(hkv, pages + 3, pr, d).transpose(0, 1)[3:]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("hkv", [1, 2])
def test_an_append_to_pools_in_one_tensor(K, bits, hkv):
    """Pools that lie in one another without sharing memory take the same bits as pools of their own; those that share it
    are refused, and may still be read."""
    from pdum_dsl_amd import _lib

    rng = np.random.default_rng(44)
    pr, d = 16, 64
    table, starts, lens, rows, pages = batch(rng, [40, 33], [40, 3], pr)
    x = torch.as_tensor(rng.standard_normal((rows, 2 * hkv, d))).bfloat16().cuda()
    k, v = x[:, :hkv], x[:, hkv:]
    t = _ints(table, starts, lens)
    own = K.paged_cache(pages, hkv, pr, d, bits=bits)
    K.paged_append(k, v, own, *t)
    for pk, pv in _layouts(pages, hkv, pr, 2 * d if bits == 16 else d // 2):
        if bits == 16:
            cache = K.PagedCache(pk.view(torch.bfloat16), pv.view(torch.bfloat16))
        else:
            scales = torch.zeros((pages, 2, hkv, pr, d // 32), dtype=torch.uint8, device="cuda")
            cache = K.PagedCache(pk, pv, scales[:, 0], scales[:, 1])
        K.paged_append(k, v, cache, *t)
        for a, b in ((cache.k, own.k), (cache.v, own.v), (cache.k_scale, own.k_scale), (cache.v_scale, own.v_scale)):
            assert a is None or torch.equal(a, b)
    if bits == 4:
        shared = (K.PagedCache(own.k, own.v, own.k_scale, own.k_scale), K.PagedCache(own.k, own.k, own.k_scale, own.v_scale))
    else:
        shared = (K.PagedCache(own.k, own.k), K.PagedCache(own.k[:1].expand(3, -1, -1, -1), own.v[:1].expand(3, -1, -1, -1)))
    for cache in shared:
        held = [p.clone() for p in (own.k, own.v)]
        with pytest.raises(_lib.PdhError, match="overlap"):
            K.paged_append(k, v, cache, *t)
        assert torch.equal(own.k, held[0]) and torch.equal(own.v, held[1])
        K.paged_rows(cache, *t, rows)
        o, _ = K.paged_attention(k, cache, *t)
        assert torch.isfinite(o.float()).all()


def test_results_in_one_tensor_with_inputs(K):
    """q's place, and other heads of the tensor that holds q, k and v, rows first and heads first; a part of q is refused."""
    from pdum_dsl_amd import _lib

    rng = np.random.default_rng(45)
    pr, d, hq, hkv = 16, 64, 4, 2
    for lengths, new in (([40, 33], [2, 1]), ([90, 33], [70, 3])):
        table, starts, lens, rows, pages = batch(rng, lengths, new, pr)
        t, tab = _ints(table, starts, lens), K.rotary_table(100, d)
        x = torch.as_tensor(rng.standard_normal((rows, 2 * hq + 2 * hkv, d))).bfloat16().cuda()
        for turned in (x, x.transpose(0, 1).contiguous().transpose(0, 1)):
            q, k, v, rest = turned[:, :hq], turned[:, hq : hq + hkv], turned[:, hq + hkv : hq + 2 * hkv], turned[:, hq + 2 * hkv :]
            want = None
            for place in (None, rest, q):
                cache, held = K.paged_cache(pages, hkv, pr, d), turned.clone()
                got = K.paged_append(k, v, cache, *t, q=q, rotary=tab, out=place).clone()
                o = K.paged_attention(q, cache, *t, out=place)[0].clone()  # (of q as it now is)
                assert want is None or torch.equal(got, want)
                want = got
                if place is None:
                    plain = o
                    assert torch.equal(turned, held)
                elif place is rest:
                    assert torch.equal(o, plain) and torch.equal(turned[:, : hq + 2 * hkv], held[:, : hq + 2 * hkv])
                else:
                    assert torch.equal(turned[:, hq:], held[:, hq:])
            turned.copy_(held)  # q as it was
        wide = torch.zeros((rows + 1, hq, d), dtype=torch.bfloat16, device="cuda")
        kv = torch.zeros((rows, hkv, d), dtype=torch.bfloat16, device="cuda")
        for q, out in ((wide[1:], wide[:-1]), (wide[:-1], wide[1:])):
            with pytest.raises(_lib.PdhError, match="overlap"):
                K.paged_append(kv, kv, cache, *t, q=q, out=out)
            with pytest.raises(_lib.PdhError, match="overlap"):
                K.paged_attention(q, cache, *t, out=out)
        with pytest.raises(_lib.PdhError, match="overlap"):
            K.paged_append(kv, wide[1:, :hkv], cache, *t, q=torch.zeros_like(wide[1:]), out=wide[1:])


@pytest.mark.parametrize("bits,gap", [(16, 14), (16, 16), (16, 17), (16, 19), (4, 16)])
@pytest.mark.parametrize("n,new,sinks,window", [(6000, 1, 0, None), (6000, 3, 0, None), (6000, 130, 0, None), (9000, 1, 1, 5000),
                                                (9000, 200, 1, 5000)])
def test_f16_weights_far_under_the_largest_still_count(K, bits, gap, n, new, sinks, window):
    """A first token takes nearly all of each row's weight, and its value is 0: the result is what thousands of weights of
    e^-gap come to. f16 has numbers down to 2^-24, and e^-17 lies under 2^-24.5."""
    rng = np.random.default_rng(46)
    pr, d, hq, hkv = 16, 64, 8, 2
    table, starts, lens, rows, pages = batch(rng, [n], [new], pr)
    x = torch.zeros((n, 2, hkv, d), dtype=torch.float16, device="cuda")
    x[0, 0, :, 0] = gap / d**-0.5  # a key whose score is gap; all others' are 0
    x[1:, 1] = torch.as_tensor(rng.choice([0.5, 1.0, 1.5, 2.0], (n - 1, hkv, d))).half()
    cache = K.paged_cache(pages, hkv, pr, d, torch.float16, bits=bits)
    K.paged_append(x[:, 0], x[:, 1], cache, *_ints(table, [0, n], lens))
    kk, vv = (_host(t) for t in K.paged_rows(cache, *_ints(table, [0, n], lens), n))
    assert (kk == _host(x[:, 0])).all() and (vv == _host(x[:, 1])).all()  # 4 bits hold these
    q = torch.zeros((rows, hq, d), dtype=torch.float16, device="cuda")
    q[:, :, 0] = 1.0
    o, lse = K.paged_attention(q, cache, *_ints(table, starts, lens), window=window, sinks=sinks)
    o, lse = _host(o), _host(lse)
    for r in range(rows):
        pos = n - new + r
        lo = 1 if window is None else pos - window + 1
        v = vv[lo : pos + 1].repeat(hq // hkv, axis=1)
        w = np.exp(-float(gap))
        den = 1 + len(v) * w
        want = w * v.sum(0) / den
        # each weight is rounded by half a step: 2^-11 of it, or of 2^-14 2^-7 where the largest is 2^7; the exponential by
        # 2^-21 and 2^-23 gap, sums by 2^-24 an addition, the result by 2^-11 or 2^-25
        part = 2.0**-11 + 2.0**-20 + gap * 2.0**-22 + len(v) * 2.0**-23
        bound = part * want + 2.0**-32 * v.sum(0)
        bound = bound + 2.0**-11 * (want + bound) + 2.0**-25
        assert (np.abs(o[r] - want) <= bound).all(), (r, np.abs(o[r] - want).max(), want.max())
        assert np.abs(lse[r] - (gap + np.log(den))).max() <= 2.0**-20 + gap * 2.0**-21 + len(v) * 2.0**-23


def test_results_between_the_pools_rows(K):
    """One tensor that holds the cache's rows and, beside them, room for results: taken, where no byte is shared."""
    from pdum_dsl_amd import _lib

    rng = np.random.default_rng(47)
    pr, d, hq, hkv, pages = 16, 64, 4, 2, 8
    table, starts, lens, rows, _ = batch(rng, [40, 33], [9, 1], pr, spare=pages - 6)
    x = torch.as_tensor(rng.standard_normal((rows, hq + 2 * hkv, d))).bfloat16().cuda()
    t = _ints(table, starts, lens)
    own = K.paged_cache(pages, hkv, pr, d)
    want = K.paged_append(x[:, hq : hq + hkv], x[:, hq + hkv :], own, *t, q=x[:, :hq])
    o, lse = K.paged_attention(want, own, *t)
    wide = torch.zeros((pages, hkv, pr, 3 * d), dtype=torch.bfloat16, device="cuda")
    cache = K.PagedCache(wide[..., :d], wide[..., d : 2 * d])
    free = wide.view(pages * hkv * pr // hq, hq, 3 * d)[:rows, :, 2 * d :]
    got = K.paged_append(x[:, hq : hq + hkv], x[:, hq + hkv :], cache, *t, q=x[:, :hq], out=free)
    assert torch.equal(got, want) and torch.equal(cache.k, own.k) and torch.equal(cache.v, own.v)
    o2, lse2 = K.paged_attention(want, cache, *t, out=free)
    assert torch.equal(o2, o) and torch.equal(lse2, lse)
    for out in (own.k.view(-1, hq, d)[:rows], own.v.view(-1, hq, d)[-rows:]):
        with pytest.raises(_lib.PdhError, match="overlap"):
            K.paged_attention(want, own, *t, out=out)
        with pytest.raises(_lib.PdhError, match="overlap"):
            K.paged_append(x[:, :hkv], x[:, :hkv], own, *t, q=want, out=out)
