"""The training operators without a GPU: the oracle's closed forms against
differences and published vectors, and every refusal of the C entry points
(each fires before any HIP call)."""

import ctypes as C

import numpy as np
import pytest

from oracle import closed_forms as cf


def test_the_generator_matches_its_published_vectors():
    # Random123's known answers for philox4x32-10
    ones = np.full((1, 4), 0xFFFFFFFF, dtype=np.uint64)
    pi = np.array([[0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344]], dtype=np.uint64)
    for ctr, key, want in (
        (np.zeros((1, 4)), (0, 0), "6627e8d5 e169c58d bc57ac4c 9b00dbd8"),
        (ones, (0xFFFFFFFF, 0xFFFFFFFF), "408f276d 41c83b0e a20bc7c6 6d5451fd"),
        (pi, (0xA4093822, 0x299F31D0), "d16cfe09 94fdcceb 5001e420 24126ea1"),
    ):
        assert " ".join(f"{int(v):08x}" for v in cf.philox4x32(ctr, key)[0]) == want


def test_the_layernorm_gradient_matches_differences():
    rng = np.random.default_rng(3)
    x, dy, g, b = (rng.standard_normal(s) for s in ((5, 11), (5, 11), 11, 11))
    dx, dg, db = cf.layernorm_bwd(x, dy, g, 1e-5)
    loss = lambda x, g, b: (dy * cf.np_layernorm(x, g, b, 1e-5)).sum()  # noqa: E731
    h = 1e-6
    for want, at in ((dx, 0), (dg, 1), (db, 2)):
        args = [x, g, b]
        v = rng.standard_normal(want.shape)
        hi, lo = list(args), list(args)
        hi[at], lo[at] = args[at] + h * v, args[at] - h * v
        # the central difference's error: h^2 of the third derivative, 2^-53 |loss| / h of rounding
        assert abs((loss(*hi) - loss(*lo)) / (2 * h) - (want * v).sum()) < 1e-7


def test_the_cross_entropy_gradient_matches_differences():
    rng = np.random.default_rng(4)
    x, w, dloss = rng.standard_normal((6, 9)), rng.standard_normal((13, 9)), rng.standard_normal(6)
    t = np.array([0, 12, -100, 5, 13, 5])  # one ignored, one past the vocabulary
    dx, dw = cf.linear_xent_bwd(x, w, t, dloss)
    h = 1e-6
    for at, want in ((0, dx), (1, dw)):
        v = rng.standard_normal(want.shape)
        f = (lambda s: (dloss * cf.linear_xent(x + s * v, w, t)[0]).sum()) if at == 0 else (
            lambda s: (dloss * cf.linear_xent(x, w + s * v, t)[0]).sum())
        assert abs((f(h) - f(-h)) / (2 * h) - (want * v).sum()) < 1e-7


FAKE = C.c_void_p(256)  # never dereferenced: every call below is refused first


def _refused(rc, text, code=None):
    from pdum_dsl_amd import _lib

    assert rc == (_lib.PDH_EINVAL if code is None else code), (rc, _lib.last_error())
    assert text in _lib.last_error(), _lib.last_error()


def test_layernorm_refusals():
    from pdum_dsl_amd import _lib

    lib = _lib.lib()

    def fwd(rows=4, cols=8, ldx=8, ldy=8, eps=1e-5, dt=1, x=FAKE):
        return lib.pdh_layernorm_fwd(x, None, None, FAKE, FAKE, FAKE, rows, cols, ldx, ldy, eps, dt, None)

    _refused(fwd(cols=0), "cols >= 1")
    _refused(fwd(rows=-1), "rows >= 0")
    _refused(fwd(ldy=7), "row strides")
    _refused(fwd(ldx=-8), "row strides")
    _refused(fwd(eps=-1.0), "eps")
    _refused(fwd(x=None), "null pointer")
    _refused(fwd(dt=7), "dtype 7", _lib.PDH_EUNSUPPORTED)
    assert fwd(rows=0) == _lib.PDH_OK

    def bwd(rows=4, cols=8, ldx=8, lddx=8, gamma=FAKE, dg=FAKE, db=FAKE, ws=FAKE, nb=1 << 20, dt=0):
        return lib.pdh_layernorm_bwd(FAKE, FAKE, None, gamma, FAKE, FAKE, FAKE, dg, db, rows, cols, ldx, 8, 0, lddx, dt,
                                     ws, nb, None)

    _refused(bwd(cols=0), "cols >= 1")
    _refused(bwd(lddx=4), "row strides")
    _refused(bwd(gamma=None), "come together")
    _refused(bwd(db=None), "come together")
    _refused(bwd(nb=4), "workspace holds 4 bytes")
    _refused(bwd(ws=None), "workspace holds 0 bytes")
    _refused(bwd(dt=3), "dtype 3", _lib.PDH_EUNSUPPORTED)
    assert lib.pdh_layernorm_bwd_workspace(0, 8, 0) == 0 and lib.pdh_layernorm_bwd_workspace(1, 8, 0) == 64


def test_dropout_refusals():
    from pdum_dsl_amd import _lib

    lib = _lib.lib()

    def drop(rows=4, cols=8, ldx=8, ldy=8, p=0.1, site=0, dt=0, rng=FAKE):
        return lib.pdh_dropout(FAKE, None, FAKE, rows, cols, ldx, 0, ldy, p, rng, site, dt, None)

    for p in (-0.1, 1.1, float("nan")):
        _refused(drop(p=p), "must lie in [0, 1]")
    _refused(drop(site=-1), "site -1")
    _refused(drop(site=1 << 32), "32 bits")
    _refused(drop(cols=0), "cols >= 1")
    _refused(drop(ldy=7), "row strides")
    _refused(drop(rng=None), "null pointer")
    _refused(drop(dt=5), "dtype 5", _lib.PDH_EUNSUPPORTED)
    assert drop(rows=0) == _lib.PDH_OK


def test_cpu_tensors_are_refused():
    torch = pytest.importorskip("torch")
    from pdum_dsl_amd import kernels as K

    x = torch.zeros(2, 8)
    for call in (
        lambda: K.layernorm_fwd(x),
        lambda: K.layernorm_bwd(x, x, x[:, 0], x[:, 0]),
        lambda: K.dropout_fwd(x, 0.1, torch.zeros(2, dtype=torch.int64)),
        lambda: K.dropout_bwd(x, 0.1, torch.zeros(2, dtype=torch.int64)),
    ):
        with pytest.raises((ValueError, RuntimeError, AssertionError)):
            call()


def test_linear_xent_refusals():
    from pdum_dsl_amd import _lib

    lib = _lib.lib()

    def fwd(n=4, d=8, v=16, ldx=8, ldw=8, dt=1, x=FAKE, ws=FAKE, nb=1 << 30):
        return lib.pdh_linear_xent_fwd(x, FAKE, FAKE, FAKE, FAKE, n, d, v, ldx, ldw, -100, dt, None, ws, nb, None)

    def bwd(n=4, d=8, v=16, ldx=8, ldw=8, dt=1, x=FAKE, ws=FAKE, nb=1 << 30):
        return lib.pdh_linear_xent_bwd(x, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, n, d, v, ldx, ldw, -100, dt, ws, nb, None)

    for f in (fwd, bwd):
        _refused(f(d=0), "width >= 1")
        _refused(f(v=0), "vocabulary >= 1")
        _refused(f(n=-1), "tokens >= 0")
        _refused(f(ldw=-8), "row strides")
        _refused(f(x=None), "null pointer")
        _refused(f(ws=None), "holds 0 bytes")
        _refused(f(nb=16), "holds 16 bytes")
        _refused(f(ws=C.c_void_p(8)), "16-byte aligned")
        _refused(f(dt=9), "dtype 9", _lib.PDH_EUNSUPPORTED)
        _refused(f(d=(1 << 18) + 1), "2^18 features", _lib.PDH_EUNSUPPORTED)
        _refused(f(n=1 << 24, v=1 << 24), "2^38 logits", _lib.PDH_EUNSUPPORTED)
    assert fwd(n=0) == _lib.PDH_OK
    _refused(bwd(n=0), "no tokens")
    need = lambda x, ldx, dt, bwd=0: lib.pdh_linear_xent_workspace(C.c_void_p(x), FAKE, 1000, 64, 5000, ldx, 64, dt, bwd)  # noqa: E731
    assert need(256, 64, 1) < need(258, 64, 1) == need(256, 65, 1) < need(256, 64, 0)  # packed where not read in place
    assert need(256, 64, 1, 1) == need(258, 64, 1, 1) < need(256, 64, 0, 1)  # the backward always packs x
    assert lib.pdh_linear_xent_workspace(FAKE, FAKE, 0, 64, 5000, 64, 64, 1, 1) == 0
