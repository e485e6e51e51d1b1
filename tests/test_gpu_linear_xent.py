"""The linear head's cross entropy and its gradient on the GPU against the
float64 closed forms.

Tolerances. u = 2^-24. An fp32 sum of k products by the matrix cores takes
k / 16 instructions of at most 4 roundings each (six times as many from split
operands): M roundings, taken as independent, are within 6 u sqrt(M) (six
standard deviations and more) of the largest partial sum, itself within |sum| +
4 sqrt(sum of squared products). So, e_z for a logit,
  |err lse|  <= e_lse = max e_z + 4 u (max|z| + |lse|) + 200 u
  |err loss| <= e_lse + e_z + u |loss|
  rel err p  <= e_p = e_z + e_lse + 4 u (|z| + |lse| + 1)
  |err dz|   <= eps/2 |dz| + |dloss| p e_p (+ fp16's subnormal spacing under its scale)
and dx, dw sum |err dz| over their products, add their own M roundings and half
a step of their type."""

import numpy as np
import pytest

from oracle import closed_forms as cf

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = 2.0**-24
HALF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _h(t):
    return t.detach().double().cpu().numpy()


def _draw(rng, shape, dtype, std=1.0):
    return torch.as_tensor(std * rng.standard_normal(shape), dtype=torch.float32).to(dtype).cuda()


def _sum_err(terms_sq, total, k, dtype):
    m = 4 * -(-k // 16) * (6 if dtype == torch.float32 else 1)
    return 6 * U * np.sqrt(m) * (np.abs(total) + 4 * np.sqrt(terms_sq))


def _bounds(x, w, t, dloss, dtype):
    z = x @ w.T
    ez = _sum_err((x**2) @ (w**2).T, z, x.shape[1], dtype)
    lse = np.log(np.exp(z - z.max(1, keepdims=True)).sum(1)) + z.max(1)
    elp = ez.max(1) + 4 * U * (np.abs(z).max(1) + np.abs(lse)) + 200 * U
    ep = ez + elp[:, None] + 4 * U * (np.abs(z) + np.abs(lse)[:, None] + 1)
    p = np.exp(z - lse[:, None])
    live = (t >= 0) & (t < w.shape[0])
    g = np.where(live, dloss, 0.0)
    hot = np.zeros_like(p)
    hot[np.nonzero(live)[0], t[live]] = 1.0
    dz = (p - hot) * g[:, None]
    edz = HALF[dtype] * np.abs(dz) + np.abs(g)[:, None] * (p * ep + 2 * U)
    if dtype == torch.float16 and np.abs(g).max() > 0:
        edz = edz + np.where(live, 2.0**-25 * 2.0 ** (np.floor(np.log2(np.abs(g).max())) + 1 - 14), 0.0)[:, None]
    dx, dw = dz @ w, dz.T @ x
    edx = edz @ np.abs(w) + _sum_err((dz**2) @ (w**2), dx, w.shape[0], dtype)
    edw = edz.T @ np.abs(x) + _sum_err((dz**2).T @ (x**2), dw, x.shape[0], dtype)
    eloss = np.where(live, elp + ez[np.arange(len(t)), np.where(live, t, 0)] + U * np.abs(lse), 0.0)
    return dict(lse=elp, loss=eloss, dx=edx, dw=edw)


def _within(got, want, bound, dtype, what):
    got = _h(got)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    lim = bound + HALF[dtype] * (np.abs(want) + bound)
    if dtype == torch.float16:
        lim = lim + 2.0**-25  # half the spacing of its subnormal values
    bad = ~(np.abs(got - want) <= lim)
    assert not bad.any(), f"{what}: {np.abs(got - want)[bad].max():.3e} past {lim[bad].min():.3e}, {bad.sum()} of {bad.size}, at {np.argwhere(bad)[0]}"


def _check(x, w, t, dloss, f, grads, dtype, ignore=None):
    hx, hw, ht, hd = _h(x).reshape(-1, x.shape[-1]), _h(w), t.cpu().numpy().reshape(-1), _h(dloss).reshape(-1)
    if ignore is not None:
        ht = np.where(ht == ignore, -1, ht)
    b = _bounds(hx, hw, ht, hd, dtype)
    loss, lse = cf.linear_xent(hx, hw, ht)
    _within(f.loss.reshape(-1), loss, b["loss"], torch.float32, "loss")
    _within(f.lse.reshape(-1), lse, b["lse"], torch.float32, "lse")
    dx, dw = cf.linear_xent_bwd(hx, hw, ht, hd)
    _within(grads[0].reshape(hx.shape), dx, b["dx"], dtype, "dx")
    _within(grads[1], dw, b["dw"], dtype, "dw")


# (tokens, width, vocab): the borders of the 256 x 128 tiles, 32-deep k tiles and 16-byte chunks
SHAPES = [(1, 1, 1), (1, 8, 2), (5, 7, 17), (33, 64, 256), (128, 32, 257), (129, 40, 255), (127, 768, 1000), (300, 100, 1003),
          (260, 33, 5003), (64, 1023, 300), (1, 768, 5003), (1000, 256, 40), (513, 264, 513)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_loss_and_gradient(shape, dtype):
    from pdum_dsl_amd import kernels as K

    n, d, v = shape
    rng = np.random.default_rng(n * 7 + d * 3 + v)
    x, w = _draw(rng, (n, d), dtype), _draw(rng, (v, d), dtype, 2.0 * d**-0.5)
    ht = rng.integers(0, v, n)
    ht[rng.random(n) < 0.1] = -100
    t = torch.as_tensor(ht).cuda()
    dloss = torch.as_tensor(rng.standard_normal(n) / n, dtype=torch.float32).cuda()
    f = K.linear_cross_entropy(x, w, t)
    g = K.linear_cross_entropy_bwd(x, w, t, f.lse, dloss)
    torch.cuda.synchronize()
    assert g[0].dtype == dtype and g[1].dtype == dtype
    _check(x, w, t, dloss, f, g, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(2100, 64, 300), (3001, 100, 203), (1600, 200, 700), (4500, 8, 9), (1030, 391, 260)])
def test_many_tokens_over_a_small_vocabulary(shape, dtype):
    """dw's product in parts over the tokens, in each width's tiles; the same bits again."""
    from pdum_dsl_amd import kernels as K

    n, d, v = shape
    rng = np.random.default_rng(n + d + v)
    x, w = _draw(rng, (n, d), dtype), _draw(rng, (v, d), dtype, 2.0 * d**-0.5)
    t = torch.as_tensor(rng.integers(0, v, n)).cuda()
    dloss = torch.as_tensor(rng.standard_normal(n) / n, dtype=torch.float32).cuda()
    f = K.linear_cross_entropy(x, w, t)
    g = K.linear_cross_entropy_bwd(x, w, t, f.lse, dloss)
    _check(x, w, t, dloss, f, g, dtype)
    for a, b in zip(g, K.linear_cross_entropy_bwd(x, w, t, f.lse, dloss)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_ignored_and_bad_targets(dtype):
    """Ignored tokens have no loss and no gradient, targets outside the
    vocabulary likewise and are counted; ignore_index may be an entry."""
    from pdum_dsl_amd import kernels as K

    rng = np.random.default_rng(2)
    n, d, v = 70, 48, 300
    x, w = _draw(rng, (n, d), dtype), _draw(rng, (v, d), dtype, 0.3)
    dloss = torch.full((n,), 1 / n, device="cuda")
    ht = rng.integers(0, v, n)
    ht[:4] = [v, -1, 2**40, -(2**62)]
    ht[4:9] = -100
    t = torch.as_tensor(ht).cuda()
    bad = torch.zeros((), dtype=torch.int32, device="cuda")
    f = K.linear_cross_entropy(x, w, t, bad=bad)
    g = K.linear_cross_entropy_bwd(x, w, t, f.lse, dloss)
    assert bad.item() == 4 and not f.loss[:9].any() and not g[0][:9].any()
    _check(x, w, t, dloss, f, g, dtype)
    some = int(ht[20])
    f = K.linear_cross_entropy(x, w, t, ignore_index=some)
    g = K.linear_cross_entropy_bwd(x, w, t, f.lse, dloss, ignore_index=some)
    assert not g[0][20].any()
    _check(x, w, t, dloss, f, g, dtype, ignore=some)
    none = torch.full((n,), -100, device="cuda")
    f = K.linear_cross_entropy(x, w, none)
    g = K.linear_cross_entropy_bwd(x, w, none, f.lse, dloss)
    assert not f.loss.any() and torch.isfinite(f.lse).all() and not g[0].any() and not g[1].any()
    zero = K.linear_cross_entropy_bwd(x, w, t, f.lse, torch.zeros_like(dloss))
    assert not zero[0].any() and not zero[1].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_and_misaligned_operands(dtype):
    """Rows of wider tensors, at chunk-aligned and odd offsets, 3-D x: as the
    contiguous call, bit for bit."""
    from pdum_dsl_amd import kernels as K

    rng = np.random.default_rng(3)
    n, d, v = 60, 72, 333
    xw, ww = _draw(rng, (n, d + 24), dtype), _draw(rng, (v, d + 40), dtype, 0.2)
    t = torch.as_tensor(rng.integers(0, v, n)).cuda()
    dloss = torch.rand(n, device="cuda")
    for ox, ow in ((8, 16), (3, 16), (8, 5), (1, 7)):
        x, w = xw[:, ox:ox + d], ww[:, ow:ow + d]
        f, fc = K.linear_cross_entropy(x, w, t), K.linear_cross_entropy(x.contiguous(), w.contiguous(), t)
        assert torch.equal(f.loss, fc.loss) and torch.equal(f.lse, fc.lse)
        g = K.linear_cross_entropy_bwd(x, w, t, f.lse, dloss)
        gc = K.linear_cross_entropy_bwd(x.contiguous(), w.contiguous(), t, f.lse, dloss)
        assert torch.equal(g[0], gc[0]) and torch.equal(g[1], gc[1])
    x3, t3 = x.contiguous().view(4, 15, d), t.view(4, 15)
    f3 = K.linear_cross_entropy(x3, w, t3)
    g3 = K.linear_cross_entropy_bwd(x3, w, t3, f3.lse, dloss.view(4, 15))
    assert f3.loss.shape == (4, 15) and torch.equal(f3.loss.view(-1), f.loss)
    assert torch.equal(g3[0].view(n, d), g[0]) and torch.equal(g3[1], g[1])
    one = x[:1].expand(n, d)  # one row for every token
    fe = K.linear_cross_entropy(one, w, t)
    assert torch.equal(fe.loss, K.linear_cross_entropy(one.contiguous(), w, t).loss)


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_logits_and_small_gradients(dtype):
    """Logits in the thousands (a probability of one), and dloss from 1e-6 to
    1e-2: fp16's dz keeps its digits under the scale."""
    from pdum_dsl_amd import kernels as K

    rng = np.random.default_rng(4)
    n, d, v = 40, 64, 500
    x, w = _draw(rng, (n, d), dtype, 20.0), _draw(rng, (v, d), dtype, 3.0)
    t = torch.as_tensor(rng.integers(0, v, n)).cuda()
    dloss = torch.as_tensor(10.0 ** rng.uniform(-6, -2, n), dtype=torch.float32).cuda()
    f = K.linear_cross_entropy(x, w, t)
    g = K.linear_cross_entropy_bwd(x, w, t, f.lse, dloss)
    _check(x, w, t, dloss, f, g, dtype)
    x, w = _draw(rng, (n, d), dtype), _draw(rng, (v, d), dtype, 0.2)
    dloss = dloss * 1e-4
    f = K.linear_cross_entropy(x, w, t)
    g = K.linear_cross_entropy_bwd(x, w, t, f.lse, dloss)
    _check(x, w, t, dloss, f, g, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_non_finite_tokens_stay_their_own(dtype):
    from pdum_dsl_amd import kernels as K

    rng = np.random.default_rng(5)
    x, w = _draw(rng, (9, 64), dtype), _draw(rng, (400, 64), dtype, 0.3)
    t = torch.as_tensor(rng.integers(0, 400, 9)).cuda()
    want = K.linear_cross_entropy(x, w, t)
    x[3, 5] = float("nan")
    x[6, 9] = float("inf")
    f = K.linear_cross_entropy(x, w, t)
    keep = [0, 1, 2, 4, 5, 7, 8]
    assert torch.equal(f.loss[keep], want.loss[keep]) and not torch.isfinite(f.loss[[3, 6]]).any()
    dx, _ = K.linear_cross_entropy_bwd(x, w, t, f.lse, torch.ones(9, device="cuda"))
    assert torch.isfinite(dx[keep]).all() and not torch.isfinite(dx[[3, 6]]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, d, v", [(40, 64, 300), (1100, 72, 333), (33, 51, 130)])
def test_ignored_tokens_may_hold_anything(n, d, v, dtype):
    """Rows of a padded batch hold NaN and infinities, as do their lse and
    dloss: the live tokens' loss and every gradient are those of finite rows."""
    from pdum_dsl_amd import kernels as K

    rng = np.random.default_rng(n)
    x, w = _draw(rng, (n, d), dtype), _draw(rng, (v, d), dtype, 0.3)
    ht = rng.integers(0, v, n)
    ht[-n // 4:] = -100
    ht[2] = v + 7
    t = torch.as_tensor(ht).cuda()
    dloss = torch.as_tensor(rng.standard_normal(n) / n, dtype=torch.float32).cuda()
    f = K.linear_cross_entropy(x, w, t)
    want = K.linear_cross_entropy_bwd(x, w, t, f.lse, dloss)
    dead = torch.as_tensor((ht < 0) | (ht >= v)).cuda()
    y, nan = x.clone(), float("nan")
    y[dead] = nan
    y[2] = float("inf")
    g = K.linear_cross_entropy(y, w, t)
    assert torch.equal(g.loss, f.loss) and torch.equal(g.lse[~dead], f.lse[~dead])
    got = K.linear_cross_entropy_bwd(y, w, t, g.lse, torch.where(dead, nan, dloss))
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_the_gradient_matches_differences():
    """Along random directions, central differences of the float64 loss."""
    from pdum_dsl_amd import kernels as K

    rng = np.random.default_rng(6)
    n, d, v = 30, 50, 200
    x, w = _draw(rng, (n, d), torch.float32), _draw(rng, (v, d), torch.float32, 0.3)
    ht = rng.integers(0, v, n)
    t = torch.as_tensor(ht).cuda()
    dloss = torch.as_tensor(rng.standard_normal(n), dtype=torch.float32).cuda()
    f = K.linear_cross_entropy(x, w, t)
    dx, dw = K.linear_cross_entropy_bwd(x, w, t, f.lse, dloss)
    hx, hw, hd = _h(x), _h(w), _h(dloss)
    b = _bounds(hx, hw, ht, hd, torch.float32)
    loss = lambda a, c: (hd * cf.linear_xent(a, c, ht)[0]).sum()  # noqa: E731
    h = 1e-5
    p, q = rng.standard_normal(hx.shape), rng.standard_normal(hw.shape)
    # the differences' own error: h^2 of the third derivative and 2^-53 |loss| / h, below 1e-6 here
    got = (_h(dx) * p).sum(), (_h(dw) * q).sum()
    want = (loss(hx + h * p, hw) - loss(hx - h * p, hw)) / (2 * h), (loss(hx, hw + h * q) - loss(hx, hw - h * q)) / (2 * h)
    assert abs(got[0] - want[0]) < 1e-6 + ((b["dx"] + U * np.abs(_h(dx))) * np.abs(p)).sum()
    assert abs(got[1] - want[1]) < 1e-6 + ((b["dw"] + U * np.abs(_h(dw))) * np.abs(q)).sum()


def test_several_pieces_of_the_vocabulary():
    """dz past one piece's bytes: against the gradient of the vocabulary's
    halves, whose sums the pieces' are (lse is the whole vocabulary's)."""
    from pdum_dsl_amd import kernels as K

    gen = torch.Generator(device="cuda").manual_seed(1)
    n, d, v = 6000, 40, 200003
    x = torch.randn((n, d), generator=gen, device="cuda").bfloat16()
    w = (0.3 * torch.randn((v, d), generator=gen, device="cuda")).bfloat16()
    t = torch.randint(0, v, (n,), generator=gen, device="cuda")
    dloss = torch.full((n,), 1.0 / n, device="cuda")
    f = K.linear_cross_entropy(x, w, t)
    dx, dw = K.linear_cross_entropy_bwd(x, w, t, f.lse, dloss)
    want_x, want_w = torch.zeros((n, d), dtype=torch.float64, device="cuda"), torch.empty((v, d), dtype=torch.float64, device="cuda")
    scale_x, scale_w = torch.zeros_like(want_x), torch.empty_like(want_w)
    for lo in range(0, v, 20000):
        wc = w[lo:lo + 20000].double()
        dz = torch.exp(x.double() @ wc.T - f.lse.double()[:, None])
        hit = (t >= lo) & (t < lo + wc.shape[0])
        dz[hit.nonzero()[:, 0], t[hit] - lo] -= 1.0
        dz /= n
        want_x += dz @ wc
        scale_x += dz.abs() @ wc.abs()
        want_w[lo:lo + 20000] = dz.T @ x.double()
        scale_w[lo:lo + 20000] = dz.abs().T @ x.double().abs()
    # dz's rounding (half a step and the logits' few units of 2^-24) over the products, and the output's rounding
    for got, want, scale in ((dx, want_x, scale_x), (dw, want_w, scale_w)):
        lim = 2.0**-8 * (want.abs() + 1.02 * scale)
        assert ((got.double() - want).abs() <= lim).all()


@pytest.mark.parametrize("n, d, v, dtype", [(3000, 200, 70001, torch.float32), (9000, 100, 70001, torch.bfloat16),
                                            (5000, 500, 120001, torch.float16)])
def test_pieces_in_every_width_of_tile(n, d, v, dtype):
    """Two pieces whose dw is in parts over the tokens (the first two shapes) or
    whole, ignored tokens among them. Against the formulas given the device's lse:
    the bounds above without lse's error."""
    from pdum_dsl_amd import kernels as K

    gen = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn((n, d), generator=gen, device="cuda").to(dtype)
    w = (0.2 * torch.randn((v, d), generator=gen, device="cuda")).to(dtype)
    t = torch.randint(0, v, (n,), generator=gen, device="cuda")
    t[::5] = -100
    g = torch.rand(n, generator=gen, device="cuda") / n
    f = K.linear_cross_entropy(x, w, t)
    dx, dw = K.linear_cross_entropy_bwd(x, w, t, f.lse, g)
    live = (t >= 0).double()[:, None]
    hx, gd, lse = x.double(), g.double()[:, None] * live, f.lse.double()[:, None]
    m = lambda k: 6 * U * (4 * -(-k // 16) * (6 if dtype == torch.float32 else 1)) ** 0.5  # noqa: E731
    tiny = 2.0**-25 * 2.0 ** (np.floor(np.log2(g.max().item())) + 1 - 14) if dtype == torch.float16 else 0.0
    wx, ex, qx = (torch.zeros((n, d), dtype=torch.float64, device="cuda") for _ in range(3))
    ok = True
    for lo in range(0, v, 10000):
        wc = w[lo:lo + 10000].double()
        z = hx @ wc.T
        ep = m(d) * (z.abs() + 4 * ((hx**2) @ (wc**2).T).sqrt()) + 4 * U * (z.abs() + lse.abs() + 1)
        p = torch.exp(z - lse)
        dz = p.clone()
        hit = (t >= lo) & (t < lo + wc.shape[0])
        dz[hit.nonzero()[:, 0], t[hit] - lo] -= 1.0
        dz *= gd
        e = HALF[dtype] * dz.abs() + gd * (p * ep + 2 * U) + tiny * live
        wx += dz @ wc
        ex += e @ wc.abs()
        qx += (dz**2) @ (wc**2)
        want = dz.T @ hx
        err = e.T @ hx.abs() + m(n) * (want.abs() + 4 * ((dz**2).T @ (hx**2)).sqrt())
        lim = err + HALF[dtype] * (want.abs() + err) + (2.0**-25 if dtype == torch.float16 else 0.0)
        ok = ok and bool(((dw[lo:lo + 10000].double() - want).abs() <= lim).all())
    assert ok
    err = ex + m(v) * (wx.abs() + 4 * qx.sqrt())
    lim = err + HALF[dtype] * (wx.abs() + err) + (2.0**-25 if dtype == torch.float16 else 0.0)
    assert ((dx.double() - wx).abs() <= lim).all()


def test_loss_repeats_and_replays_in_a_graph():
    from pdum_dsl_amd import kernels as K

    for dtype in DTYPES:
        x = torch.randn((200, 96), device="cuda").to(dtype)
        w = (0.2 * torch.randn((700, 96), device="cuda")).to(dtype)
        t = torch.randint(0, 700, (200,), device="cuda")
        dloss = torch.full((200,), 1 / 200, device="cuda")

        def step():
            f = K.linear_cross_entropy(x, w, t)
            return (f.loss, f.lse) + K.linear_cross_entropy_bwd(x, w, t, f.lse, dloss)

        a, b = step(), step()
        assert all(torch.equal(p, q) for p, q in zip(a, b))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        for _ in range(3):
            x.copy_(torch.randn((200, 96), device="cuda"))
            t.copy_(torch.randint(0, 700, (200,), device="cuda"))
            want = step()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_loss_refusals_and_no_tokens():
    from pdum_dsl_amd import kernels as K
    from pdum_dsl_amd._lib import PdhError

    x, w = torch.randn((4, 8), device="cuda"), torch.randn((10, 8), device="cuda")
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    f = K.linear_cross_entropy(x, w, t)
    for call, text in (
        (lambda: K.linear_cross_entropy(x.double(), w, t), "one element type"),
        (lambda: K.linear_cross_entropy(x, w.half(), t), "one element type"),
        (lambda: K.linear_cross_entropy(x, w[:, :7], t), "width"),
        (lambda: K.linear_cross_entropy(x, w[:0], t), "vocab"),
        (lambda: K.linear_cross_entropy(x, w, t[:3]), "targets must be"),
        (lambda: K.linear_cross_entropy(x, w, t.int()), "targets must be"),
        (lambda: K.linear_cross_entropy(x, w, t.cpu()), "device tensors"),
        (lambda: K.linear_cross_entropy(x, w, t, bad=torch.zeros(1, device="cuda")), "int32"),
        (lambda: K.linear_cross_entropy_bwd(x, w, t, f.lse[:3], f.loss), "lse must be"),
        (lambda: K.linear_cross_entropy_bwd(x, w, t, f.lse, f.loss.double()), "dloss must be"),
    ):
        with pytest.raises(ValueError, match=text):
            call()
    with pytest.raises(PdhError, match="2.18 features"):
        big = torch.empty((1, (1 << 18) + 1), device="cuda")
        K.linear_cross_entropy(big, big, t[:1])
    e = torch.empty((0, 8), device="cuda")
    f = K.linear_cross_entropy(e, w, t[:0])
    dx, dw = K.linear_cross_entropy_bwd(e, w, t[:0], f.lse, f.lse)
    assert f.loss.shape == (0,) and dx.shape == (0, 8) and dw.shape == w.shape and not dw.any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_equal_weights_leave_no_common_rounding_error(dtype):
    """A mean's weights all lie half a step between two 16-bit values: held to
    them, every target's entry of dz would err by the same eps / 2, which no sum
    averages out. dz's other terms are small here, so the gradients' error is the
    rounding of the outputs, and half as much again at most."""
    from pdum_dsl_amd import kernels as K

    rng = np.random.default_rng(12)
    n, d, v = 400, 256, 3000
    x, w = _draw(rng, (n, d), dtype), _draw(rng, (v, d), dtype, 2.0 * d**-0.5)
    ht = rng.integers(0, v, n)
    t = torch.as_tensor(ht).cuda()
    weight = (1.0 + HALF[dtype]) * 2.0**-8
    dloss = torch.full((n,), weight, device="cuda")
    f = K.linear_cross_entropy(x, w, t)
    got = K.linear_cross_entropy_bwd(x, w, t, f.lse, dloss)
    for a, want in zip(got, cf.linear_xent_bwd(_h(x), _h(w), ht, np.full(n, weight))):
        rounded = _h(torch.as_tensor(want).to(dtype))
        assert np.linalg.norm(_h(a) - want) <= 1.5 * np.linalg.norm(rounded - want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,d,v", [(5, 64, 17), (131, 72, 300), (1, 40, 1), (70, 33, 129)])
@pytest.mark.parametrize("shift", [0, 1])
def test_nothing_beside_the_operands_is_read(n, d, v, dtype, shift):
    """x, w and the workspace lie in memory full of NaN (what a tile reads past
    its operand has to count as zero), at whole chunks and one element on: the
    results are those of operands that stand alone, and nothing is written
    beside the outputs."""
    from pdum_dsl_amd import _lib
    from pdum_dsl_amd import kernels as K

    rng = np.random.default_rng(n + d + v)
    x, w = _draw(rng, (n, d), dtype), _draw(rng, (v, d), dtype, 0.3)
    t = torch.as_tensor(rng.integers(0, v, n)).cuda()
    dloss = torch.as_tensor(rng.standard_normal(n), dtype=torch.float32).cuda()
    f = K.linear_cross_entropy(x, w, t)
    want = K.linear_cross_entropy_bwd(x, w, t, f.lse, dloss)

    def within(a):
        big = torch.full((a.shape[0] + 1024, a.shape[1] + 64), float("nan"), dtype=dtype, device="cuda")
        view = big[512:512 + a.shape[0], 16 + shift:16 + shift + a.shape[1]]
        view.copy_(a)
        return view

    bx, bw = within(x), within(w)
    f2 = K.linear_cross_entropy(bx, bw, t)
    assert torch.equal(f.loss, f2.loss) and torch.equal(f.lse, f2.lse)
    lib, code, sizes = _lib.lib(), K._DT[dtype], (n, d, v, bx.stride(0), bw.stride(0))
    need = lib.pdh_linear_xent_workspace(bx.data_ptr(), bw.data_ptr(), *sizes, code, 1)
    ws = torch.full((need + 4096,), 255, dtype=torch.uint8, device="cuda")
    out = [torch.full((a.shape[0] + 2, a.shape[1]), 7.0, dtype=dtype, device="cuda") for a in want]
    _lib.call("pdh_linear_xent_bwd", bx.data_ptr(), bw.data_ptr(), t.data_ptr(), f.lse.data_ptr(), dloss.data_ptr(),
              out[0][1:].data_ptr(), out[1][1:].data_ptr(), *sizes, -100, code, ws.data_ptr(), need, K._stream())
    torch.cuda.synchronize()
    for a, b in zip(out, want):
        assert torch.equal(a[1:-1], b) and (a[0] == 7).all() and (a[-1] == 7).all()
    assert (ws[need:] == 255).all()


def test_one_token_alone_and_numpy_scalars():
    from pdum_dsl_amd import kernels as K

    x, w = torch.randn(48, device="cuda"), torch.randn((30, 48), device="cuda")
    t = torch.tensor(7, device="cuda")
    f = K.linear_cross_entropy(x, w, t, ignore_index=np.int64(-100))
    dx, dw = K.linear_cross_entropy_bwd(x, w, t, f.lse, torch.ones((), device="cuda"), ignore_index=np.int32(-100))
    g = K.linear_cross_entropy(x[None], w, t[None])
    assert f.loss.shape == () and dx.shape == (48,) and dw.shape == (30, 48) and torch.equal(f.loss, g.loss[0])
    r = torch.tensor([1, 2], device="cuda")
    assert torch.equal(K.dropout_fwd(x, np.float32(0.5), r, site=np.int64(1)), K.dropout_fwd(x, 0.5, r, site=1))
    assert torch.equal(K.layernorm_fwd(x, eps=np.float64(1e-5)).y, K.layernorm_fwd(x[None]).y[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [1e-30, 1e30])
def test_weights_of_any_size(dtype, size):
    """dloss as small or large as fp32 allows: dx and dw are those of weights near one, times it (in fp32's range,
    and in bf16's; fp16's output range ends first)."""
    from pdum_dsl_amd import kernels as K

    rng = np.random.default_rng(9)
    x, w = _draw(rng, (60, 64), dtype), _draw(rng, (200, 64), dtype, 0.3)
    t = torch.as_tensor(rng.integers(0, 200, 60)).cuda()
    weight = torch.as_tensor(rng.random(60) + 0.5, dtype=torch.float32).cuda()
    f = K.linear_cross_entropy(x, w, t)
    one = K.linear_cross_entropy_bwd(x, w, t, f.lse, weight)
    got = K.linear_cross_entropy_bwd(x, w, t, f.lse, weight * size)
    if dtype == torch.float16:
        assert all((g == 0).all() if size < 1 else torch.isinf(g[o.abs() > 1e-3]).all() for g, o in zip(got, one))
        return
    for g, o in zip(got, one):  # each rounded once from sums over weights that differ in their last place
        assert ((g.double() / size - o.double()).abs() <= 4 * HALF[dtype] * o.double().abs() + 1e-6 * o.double().abs().max()).all()
