"""The paged-cache operators without a GPU: the oracle against independent
forms, and every refusal of the C entry points and of the wrappers (each fires
before any HIP call)."""

import ctypes as C

import numpy as np
import pytest

from oracle import paged as op


def test_the_rotation_keeps_lengths_and_depends_on_distances():
    rng = np.random.default_rng(0)
    tab = op.rotary_table(300, 64)
    q, k = rng.standard_normal((2, 1, 64))
    for inter in (False, True):
        dots = []
        for p, s in ((10, 3), (207, 200), (299, 292)):
            a, b = op.rotate(q, tab[p], inter), op.rotate(k, tab[s], inter)
            # 64 products of numbers turned in fp32: each off by 3 roundings, the table by one more
            assert abs(np.linalg.norm(a) - np.linalg.norm(q)) < 64 * 2.0**-22 * np.linalg.norm(q)
            dots.append(float((a.astype(np.float64) @ b.T.astype(np.float64))[0, 0]))
        # equal distances, equal products; the table's entries are rounded to fp32
        assert max(dots) - min(dots) < 64 * 2.0**-22 * np.linalg.norm(q) * np.linalg.norm(k)
        assert np.array_equal(op.rotate(q, tab[0], inter), q.astype(np.float32))


def test_four_bits_are_never_half_a_step_off():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((40, 64)) * 10.0 ** rng.integers(-6, 6, (40, 1))
    codes, scale = op.fp4(x, 125)
    got = op.fp4_values(codes, scale)
    unit = np.repeat(2.0 ** (scale.astype(float) - 127), 32, axis=-1)
    a = np.abs(x) / unit
    step = np.where(a <= 2, 0.5, np.where(a <= 4, 1.0, 2.0))
    assert (np.abs(got - x) <= 0.5 * step * unit * (1 + 2.0**-50)).all()
    top = np.abs(x).reshape(40, 2, 32).max(-1)
    assert (top <= 7 * 2.0 ** (scale - 127.0)).all() and (top > 3.5 * 2.0 ** (scale - 127.0)).all()


def test_the_oracle_is_softmax_attention():
    """Whole prompts of one sequence against a masked softmax over a dense matrix."""
    rng = np.random.default_rng(2)
    n, d, hq, hkv, pr = 37, 8, 4, 2, 16
    table = np.array([[2, 0, 1]])
    k, v = rng.standard_normal((2, 3, hkv, pr, d))
    q = rng.standard_normal((n, hq, d))
    o, lse, *_ = op.attention(q, k, v, table, [0, n], [n], scale=0.3, window=9, sinks=2)
    for h in range(hq):
        kk, vv = (x[table[0], h // 2].reshape(-1, d)[:n] for x in (k, v))
        z = 0.3 * q[:, h] @ kk.T
        t, s = np.arange(n)[:, None], np.arange(n)
        z = np.where((s <= t) & ((s > t - 9) | (s < 2)), z, -np.inf)
        p = np.exp(z)
        np.testing.assert_allclose(o[:, h], p @ vv / p.sum(1, keepdims=True), rtol=1e-12, atol=1e-14)
        np.testing.assert_allclose(lse[:, h], np.log(p.sum(1)), rtol=1e-12)


FAKE = 256  # a pointer that is never dereferenced: every call below is refused first


def _structs(cache=None, batch=None):
    from pdum_dsl_amd import _lib

    c = _lib.PagedCacheC(FAKE, FAKE, None, None, 4, 2, 16, 64, 2048, 1024, 64, 0, 0, 0, _lib.PDH_BF16, 16)
    b = _lib.PagedBatch(FAKE, FAKE, FAKE, 3, 5, 4, 4)
    for st, changes in ((c, cache), (b, batch)):
        for n, v in (changes or {}).items():
            setattr(st, n, v)
    return c, b


def _four_bits(**kw):
    return dict(bits=4, k_scale=FAKE, v_scale=FAKE, ssr=2, sr=32, **kw)


def _calls(c, b):
    from pdum_dsl_amd import _lib

    lib, p = _lib.lib(), C.c_void_p(FAKE)
    yield lib.pdh_paged_append(p, p, p, p, 4, 256, 64, 256, 64, 256, 64, 256, 64, C.byref(c), C.byref(b), None, 0, 0, 0,
                               0, 1, None, None)
    yield lib.pdh_paged_rows(p, p, 128, 64, 128, 64, C.byref(c), C.byref(b), 1, None)
    yield lib.pdh_paged_attention(p, p, None, 4, 256, 64, 256, 64, C.byref(c), C.byref(b), 1 << 40, 0, 1.0, 1, p, 1 << 40,
                                  None)


@pytest.mark.parametrize("cache,batch,text,code", [
    (dict(dtype=0), None, "dtype must be bf16 or f16", "U"),
    (dict(bits=8), None, "16 or 4 bits", "U"),
    (dict(features=96), None, "features must be 64 or 128", "U"),
    (dict(page_rows=24), None, "power of two", "U"),
    (dict(page_rows=8), None, "power of two", "U"),
    (dict(page_rows=8192), None, "power of two", "U"),
    (dict(pages=0), None, "number of pages", "E"),
    (dict(heads=0), None, "number of pages or heads", "E"),
    (dict(k=None), None, "pools", "E"),
    (dict(v=FAKE + 8), None, "16-byte aligned", "E"),
    (dict(sp=-8), None, "strides", "E"),
    (dict(sh=1028), None, "multiples of 16 bytes", "E"),
    (dict(sr=56), None, "rows overlap", "E"),
    (dict(sr=1 << 16), None, "2^16", "E"),
    (_four_bits(sp=8), None, "multiples of 16 bytes", "E"),
    (dict(_four_bits(), k_scale=None), None, "needs its scales", "E"),
    (dict(_four_bits(), ssr=1), None, "scales' rows", "E"),
    (dict(sp=1 << 34), None, "2^35 bytes", "E"),
    (_four_bits(ssp=1 << 31), None, "2^31 bytes", "E"),
    (dict(_four_bits(), ssp=-1), None, "scales' strides", "E"),
    (None, dict(rows=1 << 24), "rows", "E"),
    (None, dict(rows=-1), "rows", "E"),
    (None, dict(seqs=(1 << 20) + 1), "sequences", "E"),
    (None, dict(width=1 << 27), "2^30 tokens", "E"),
    (None, dict(table=None), "null table", "E"),
    (None, dict(lengths=None), "null table", "E"),
])
def test_refusals_of_a_cache_and_a_batch(cache, batch, text, code):
    from pdum_dsl_amd import _lib

    c, b = _structs(cache, batch)
    for rc in _calls(c, b):
        assert rc == (_lib.PDH_EUNSUPPORTED if code == "U" else _lib.PDH_EINVAL), (rc, _lib.last_error())
        assert text in _lib.last_error(), _lib.last_error()


def test_refusals_of_each_call():
    from pdum_dsl_amd import _lib

    lib, p = _lib.lib(), C.c_void_p(FAKE)
    c, b = _structs()

    def append(k=p, q=p, out=p, hq=4, k_st=256, q_sh=64, rot=None, n=0, rotated=0, ld=0):
        return lib.pdh_paged_append(k, p, q, out, hq, k_st, 64, 256, 64, 256, q_sh, 256, 64, C.byref(c), C.byref(b), rot, n,
                                    rotated, ld, 0, 1, None, None)

    def attend(q=p, o=p, hq=4, q_st=256, window=5, sinks=0, scale=1.0, ws=p, n=1 << 40, cc=c):
        return lib.pdh_paged_attention(q, o, None, hq, q_st, 64, 256, 64, C.byref(cc), C.byref(b), window, sinks, scale, 1,
                                       ws, n, None)

    bad = [
        (append(k=None), "k, v, q and q_out"), (append(out=None), "come together"), (append(hq=0), "come together"),
        (append(k_st=252), "strides"), (append(q_sh=-64), "strides"), (append(rot=p, n=9, rotated=24, ld=24), "rotated"),
        (append(rot=p, n=9, rotated=80, ld=80), "rotated"), (append(rot=p, n=9, rotated=32, ld=16), "rotary"),
        (attend(q=None), "q and o"), (attend(o=C.c_void_p(FAKE + 2)), "16-byte"), (attend(hq=3), "multiple"),
        (attend(hq=0), "multiple"), (attend(q_st=4), "strides"), (attend(window=0), "window"), (attend(sinks=-1), "sinks"),
        (attend(scale=0.0), "scale"), (attend(scale=float("nan")), "scale"), (attend(scale=float("inf")), "scale"),
        (lib.pdh_paged_rows(None, p, 128, 64, 128, 64, C.byref(c), C.byref(b), 1, None), "outputs"),
        (lib.pdh_paged_rows(p, p, 100, 64, 128, 64, C.byref(c), C.byref(b), 1, None), "strides"),
        (lib.pdh_paged_rows(p, p, 128, 64, 128, 64, None, C.byref(b), 1, None), "null cache"),
    ]
    assert all(rc in (_lib.PDH_EINVAL, _lib.PDH_EUNSUPPORTED) for rc, _ in bad), bad
    for call, text in (
        (lambda: append(k=None), "k, v, q and q_out"), (lambda: append(hq=0), "come together"),
        (lambda: attend(scale=-1.0), "scale must be finite"), (lambda: attend(hq=3), "multiple of the cache's heads"),
    ):
        assert call() == _lib.PDH_EINVAL and text in _lib.last_error(), _lib.last_error()
    # nothing to do is done without a device
    c, b = _structs(None, dict(rows=0))
    assert append() == _lib.PDH_OK and attend() == _lib.PDH_OK


def test_wrapper_refusals():
    torch = pytest.importorskip("torch")
    from pdum_dsl_amd import kernels as K

    z = lambda *s, dt=torch.bfloat16: torch.zeros(s, dtype=dt)  # noqa: E731
    u8 = torch.uint8
    for cache, text in (
        (K.PagedCache(z(2, 2, 16, 64, dt=torch.float32), z(2, 2, 16, 64, dt=torch.float32)), "bf16 or f16"),
        (K.PagedCache(z(2, 2, 16, 64), z(2, 2, 16, 64, dt=torch.float16)), "k and v are both"),
        (K.PagedCache(z(2, 2, 16, 64), z(2, 2, 16, 64), dtype=torch.float16), "k and v are both"),
        (K.PagedCache(z(2, 2, 16, 64), z(2, 1, 16, 64)), "page_rows, features"),
        (K.PagedCache(z(0, 2, 16, 64), z(0, 2, 16, 64)), "not empty"),
        (K.PagedCache(z(2, 2, 64, 16).transpose(2, 3), z(2, 2, 16, 64)), "contiguous"),
        (K.PagedCache(z(2, 2, 16, 64), z(2, 16, 2, 64).transpose(1, 2)), "same strides"),
        (K.PagedCache(z(2, 2, 16, 32, dt=u8), z(2, 2, 16, 32, dt=u8)), "k_scale and v_scale"),
        (K.PagedCache(z(2, 2, 16, 64), z(2, 2, 16, 64), z(2, 2, 16, 2, dt=u8), None), "k_scale and v_scale"),
        (K.PagedCache(z(2, 2, 16, 32, dt=u8), z(2, 2, 16, 32, dt=u8), z(2, 2, 16, 1, dt=u8), z(2, 2, 16, 2, dt=u8)),
         "k_scale must be"),
    ):
        with pytest.raises(ValueError, match=text):
            cache.c
    with pytest.raises(ValueError, match="16 or 4 bits"):
        K.paged_cache(2, 2, 16, 64, bits=8, device="cpu")
    cache = K.paged_cache(2, 2, 16, 64, bits=4, device="cpu")
    assert cache.c.bits == 4 and cache.c.features == 64 and cache.k.shape == (2, 2, 16, 32)
    i32 = torch.int32
    t = (z(1, 2, dt=i32), z(2, dt=i32), z(1, dt=i32))
    with pytest.raises(ValueError, match="CPU tensor"):
        K.paged_attention(z(1, 2, 64), cache, *t)
    with pytest.raises(ValueError, match="CPU tensor"):
        K.paged_append(z(1, 2, 64), z(1, 2, 64), cache, *t)
    # the shapes, without a device to be on
    def batch(table, starts, lengths, others=()):
        real = K._one_device
        K._one_device = lambda *ts: None
        try:
            return K._paged("f", cache, table, starts, lengths, 1, others)
        finally:
            K._one_device = real

    assert batch(*t).width == 2
    for bad in ((t[0].long(), t[1], t[2]), (t[0], t[1][:1], t[2]), (z(2, 2, dt=i32), t[1], t[2]),
                (t[0], t[1], z(1, 1, dt=i32)), (z(1, 4, dt=i32)[:, ::2], t[1], t[2])):
        with pytest.raises(ValueError):
            batch(*bad)
    with pytest.raises(ValueError, match="features must be contiguous"):
        K._tokens("f", "q", z(3, 64, 2).transpose(1, 2), torch.bfloat16, 2, 64)
    with pytest.raises(ValueError, match="must be"):
        K._tokens("f", "q", z(3, 2, 64), torch.float16, 2, 64)
    with pytest.raises(ValueError, match="overlap"):
        K._written("f", "out", z(1, 2, 64).expand(3, 2, 64))
    K._written("f", "out", z(2, 3, 64).transpose(0, 1))


def test_sizes_past_a_launch_and_sums_past_64_bits():
    from pdum_dsl_amd import _lib

    lib, p = _lib.lib(), C.c_void_p(FAKE)
    c, b = _structs(dict(heads=64, sp=64 * 16 * 64), dict(seqs=1 << 20, rows=(1 << 24) - 1))

    def attend(window=5, sinks=0, scale=1.0):
        return lib.pdh_paged_attention(p, p, None, 128, 128 * 64, 64, 128 * 64, 64, C.byref(c), C.byref(b), window, sinks,
                                       scale, 1, p, 1 << 40, None)

    assert attend() == _lib.PDH_EINVAL and "workgroups" in _lib.last_error(), _lib.last_error()
    assert attend(scale=3.0e38) == _lib.PDH_EINVAL and "scale" in _lib.last_error()  # scale log2 e is past fp32
    most = (1 << 63) - 1
    c, b = _structs(None, dict(rows=200, seqs=1, width=1 << 20))
    size = lambda window, sinks: lib.pdh_paged_attention_workspace(C.byref(c), C.byref(b), 4, window, sinks)  # noqa: E731
    assert size(most, 0) == size(1, most) == size(most, most) > size(5, 0)
