"""Layer norm's training forward and backward and the counter-based dropout on
the GPU against the float64 closed forms.

Tolerances, in units u = 2^-24 of fp32 arithmetic plus half a step of the
storage type (eps / 2 relative). A row's sum takes at most 16 additions in a
lane, 4 rotations, 2 joins and 16 waves (38; 1024-lane long rows of up to
20000 columns 20 + 6 + 16): N = 44 roundings, so
  |err mean| <= N u mean|x|, rel err rstd <= (N + 6) / 2 u + (err mean)^2 (negligible)
  |err xh| <= e_xh = u (rstd (N mean|x| + |x - mean| + |x|) + N |xh|)
  |err y|  <= |gamma| e_xh + 3 u (|xh gamma| + |beta|)
  |err dx| <= rstd [ 6 u (|u_| + |c1| + |xh c2|) + N u (mean|u_| + |xh| mean|u_ xh|) + e_xh |c2| + |xh| mean(|u_| e_xh) ] + N u |dx|
and the weights' sums take at most rows / 512 + 4 + 64 + 8 + 64 < 160 additions
for the sizes here: |err dgamma| <= 160 u sum|dy xh| + sum|dy| e_xh."""

import numpy as np
import pytest

from oracle import closed_forms as cf

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = 2.0**-24
N = 44
HALF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _h(t):
    return t.detach().double().cpu().numpy()


def _draw(rng, shape, dtype, std=1.0, mean=0.0):
    return torch.as_tensor(mean + std * rng.standard_normal(shape), dtype=torch.float32).to(dtype).cuda()


def _within(got, want, bound, dtype, what):
    got = _h(got)
    lim = bound + HALF[dtype] * (np.abs(want) + bound)
    if dtype == torch.float16:
        lim = lim + 2.0**-25  # half the spacing of its subnormal values
    bad = ~(np.abs(got - want) <= lim)
    assert not bad.any(), f"{what}: {np.abs(got - want)[bad].max():.3e} past {lim[bad].min():.3e} at {np.argwhere(bad)[0]}"


def _norm_bounds(x, g, b, dy=None, eps=1e-5):
    n = x.shape[-1]
    mu = x.mean(-1, keepdims=True)
    rstd = 1 / np.sqrt(((x - mu) ** 2).mean(-1, keepdims=True) + eps)
    xh = (x - mu) * rstd
    m1 = lambda a: np.abs(a).mean(-1, keepdims=True)  # noqa: E731
    exh = U * (rstd * (N * m1(x) + np.abs(x - mu) + np.abs(x)) + N * np.abs(xh))
    ga = np.ones(n) if g is None else np.abs(g)
    ey = ga * exh + 3 * U * (np.abs(xh) * ga + (0 if b is None else np.abs(b)))
    out = dict(mean=N * U * m1(x)[..., 0], rstd=(N + 6) * U * rstd[..., 0] + U * rstd[..., 0] ** 2 * N * m1(x)[..., 0], y=ey)
    if dy is not None:
        u = dy * (1 if g is None else g)
        c1, c2 = u.mean(-1, keepdims=True), (u * xh).mean(-1, keepdims=True)
        dx = rstd * (u - c1 - xh * c2)
        out["dx"] = rstd * (6 * U * (np.abs(u) + np.abs(c1) + np.abs(xh * c2)) + N * U * (m1(u) + np.abs(xh) * m1(u * xh))
                            + exh * np.abs(c2) + np.abs(xh) * (np.abs(u) * exh).mean(-1, keepdims=True)) + N * U * np.abs(dx)
        flat = lambda a: np.abs(a).reshape(-1, n)  # noqa: E731
        out["dgamma"] = 160 * U * flat(dy * xh).sum(0) + (flat(dy) * flat(exh)).sum(0)
        out["dbeta"] = 160 * U * flat(dy).sum(0)
    return out


# every wave count and its borders, odd widths, one column, one row, rows past a pass of the backward's grid
SHAPES = [(1, 1), (3, 5), (1, 768), (64, 768), (5, 1023), (2500, 100), (4, 1024), (7, 1025), (3, 4096), (2, 4097), (600, 2051),
          (3, 8192), (2, 8193), (2, 16384), (2, 16385), (70, 20001)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_layernorm_forward_and_backward(shape, dtype):
    from pdum_dsl_amd import kernels as K

    rng = np.random.default_rng(shape[0] * 31 + shape[1])
    n = shape[1]
    x, dy, dres = _draw(rng, shape, dtype, 1.5, 0.5), _draw(rng, shape, dtype), _draw(rng, shape, dtype)
    g, b = _draw(rng, n, dtype, 0.3, 1.0), _draw(rng, n, dtype, 0.3)
    f = K.layernorm_fwd(x, g, b, 1e-5)
    dx, dg, db = K.layernorm_bwd(x, dy, f.mean, f.rstd, g, dres=dres)
    torch.cuda.synchronize()
    hx, hdy, hg, hb, hr = _h(x), _h(dy), _h(g), _h(b), _h(dres)
    bd = _norm_bounds(hx, hg, hb, hdy)
    _within(f.mean, hx.mean(-1), bd["mean"], torch.float32, "mean")
    _within(f.rstd, 1 / np.sqrt(hx.var(-1) + 1e-5), bd["rstd"], torch.float32, "rstd")
    _within(f.y, cf.np_layernorm(hx, hg, hb), bd["y"], dtype, "y")
    wx, wg, wb = cf.layernorm_bwd(hx, hdy, hg, 1e-5, hr)
    _within(dx, wx, bd["dx"] + 2 * U * (np.abs(wx) + np.abs(hr)), dtype, "dx")
    _within(dg, wg, bd["dgamma"], dtype, "dgamma")
    _within(db, wb, bd["dbeta"], dtype, "dbeta")


@pytest.mark.parametrize("dtype", DTYPES)
def test_layernorm_without_weights_and_over_strided_rows(dtype):
    """No gamma: no weights' gradients. Rows of a wider tensor at odd element
    offsets, 3-D shapes, a broadcast dy: as the contiguous call, bit for bit."""
    from pdum_dsl_amd import kernels as K

    rng = np.random.default_rng(5)
    wide, widey = _draw(rng, (37, 211), dtype), _draw(rng, (37, 223), dtype)
    x, dy = wide[:, 3:204], widey[:, 5:206]
    f, fc = K.layernorm_fwd(x), K.layernorm_fwd(x.contiguous())
    assert all(torch.equal(a, b) for a, b in ((f.y, fc.y), (f.mean, fc.mean), (f.rstd, fc.rstd)))
    dx, dg, db = K.layernorm_bwd(x, dy, f.mean, f.rstd)
    assert dg is None and db is None
    hx, hdy = _h(x), _h(dy)
    bd = _norm_bounds(hx, None, None, hdy)
    _within(f.y, cf.np_layernorm(hx), bd["y"], dtype, "y")
    _within(dx, cf.layernorm_bwd(hx, hdy)[0], bd["dx"], dtype, "dx")
    g = _draw(rng, 201, dtype)
    one = K.layernorm_bwd(x, dy, f.mean, f.rstd, g)
    two = K.layernorm_bwd(x.contiguous(), dy.contiguous(), f.mean, f.rstd, g)
    assert all(torch.equal(a, b) for a, b in zip(one, two))
    row = dy[:1]
    one = K.layernorm_bwd(x, row.expand(37, 201), f.mean, f.rstd, g)
    two = K.layernorm_bwd(x, row.repeat(37, 1), f.mean, f.rstd, g)
    assert all(torch.equal(a, b) for a, b in zip(one, two))
    x3 = x.contiguous()[:36].reshape(4, 9, 201)
    f3 = K.layernorm_fwd(x3, g)
    assert f3.mean.shape == (4, 9) and torch.equal(f3.y.reshape(36, 201), K.layernorm_fwd(x[:36], g).y)
    perm = x3.transpose(0, 1)  # leading dims that do not compose: copied
    assert torch.equal(K.layernorm_fwd(perm, g).y, f3.y.transpose(0, 1))


def test_layernorm_zero_rows_constant_rows_and_non_finite_rows():
    from pdum_dsl_amd import kernels as K

    e = torch.empty((0, 16), device="cuda")
    g = torch.ones(16, device="cuda")
    f = K.layernorm_fwd(e, g)
    dx, dg, db = K.layernorm_bwd(e, e, f.mean, f.rstd, g)
    assert f.y.shape == (0, 16) and dx.shape == (0, 16) and not dg.any() and not db.any()
    x = torch.randn((6, 50), device="cuda")
    x[1] = 3.0  # no variance: rstd = eps^-1/2
    x[3, 7] = float("inf")
    x[4, 49] = float("nan")
    gg = torch.ones(50, device="cuda")
    f = K.layernorm_fwd(x, gg, None, 1e-5)
    dx, dg, _ = K.layernorm_bwd(x, torch.ones_like(x), f.mean, f.rstd, gg)
    assert torch.equal(f.y[1], torch.zeros(50, device="cuda")) and abs(f.rstd[1].item() - 1e-5**-0.5) < 1e-4
    for t in (f.y, dx):
        assert torch.isfinite(t[[0, 1, 2, 5]]).all() and torch.isnan(t[3]).any() and torch.isnan(t[4]).all()


def test_layernorm_in_place_and_repeatable():
    from pdum_dsl_amd import kernels as K

    x = torch.randn((333, 1000), device="cuda", dtype=torch.bfloat16)
    dy, g = torch.randn_like(x), torch.randn(1000, device="cuda", dtype=torch.bfloat16)
    f = K.layernorm_fwd(x, g)
    a = K.layernorm_bwd(x, dy, f.mean, f.rstd, g)
    b = K.layernorm_bwd(x, dy, f.mean, f.rstd, g)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    z = x.clone()
    assert K.layernorm_fwd(z, g, out=z).y is z and torch.equal(z, f.y)


@pytest.mark.parametrize("where", ["x", "dy", "dres"])
@pytest.mark.parametrize("cols", [3, 100, 1500, 5000, 9001, 16401])
def test_layernorm_gradient_in_the_place_of_an_input(cols, where):
    """The C entry point's dx may be x, dy or dres: as into a tensor of its own, bit for bit."""
    from pdum_dsl_amd import _lib
    from pdum_dsl_amd import kernels as K

    rows = 37
    ins = {k: torch.randn((rows, cols), device="cuda").bfloat16() for k in ("x", "dy", "dres")}
    g = torch.randn(cols, device="cuda").bfloat16()
    f = K.layernorm_fwd(ins["x"], g)
    want = K.layernorm_bwd(ins["x"], ins["dy"], f.mean, f.rstd, g, dres=ins["dres"])
    dg, db = torch.empty_like(g), torch.empty_like(g)
    need = _lib.lib().pdh_layernorm_bwd_workspace(rows, cols, _lib.PDH_BF16)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    _lib.call("pdh_layernorm_bwd", ins["x"].data_ptr(), ins["dy"].data_ptr(), ins["dres"].data_ptr(), g.data_ptr(),
              f.mean.data_ptr(), f.rstd.data_ptr(), ins[where].data_ptr(), dg.data_ptr(), db.data_ptr(), rows, cols,
              cols, cols, cols, cols, _lib.PDH_BF16, ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    for a, b in zip((ins[where], dg, db), want):
        assert torch.equal(a, b)


def test_layernorm_gradient_matches_differences():
    """The device's gradient against central differences of the float64
    forward along random directions."""
    from pdum_dsl_amd import kernels as K

    rng = np.random.default_rng(8)
    x, dy, g = (_draw(rng, s, torch.float32) for s in ((20, 130), (20, 130), 130))
    f = K.layernorm_fwd(x, g)
    dx, dg, _ = K.layernorm_bwd(x, dy, f.mean, f.rstd, g)
    hx, hdy, hg = _h(x), _h(dy), _h(g)
    bd = _norm_bounds(hx, hg, None, hdy)
    h = 1e-5
    v, w = rng.standard_normal(hx.shape), rng.standard_normal(130)
    loss = lambda a, b: (hdy * cf.np_layernorm(a, b)).sum()  # noqa: E731
    # the difference's own error is below 1e-7 (h^2 of the third derivative, 2^-53 |loss| / h)
    assert abs((loss(hx + h * v, hg) - loss(hx - h * v, hg)) / (2 * h) - (_h(dx) * v).sum()) < 1e-6 + (
        (bd["dx"] + U * np.abs(_h(dx))) * np.abs(v)).sum()
    assert abs((loss(hx, hg + h * w) - loss(hx, hg - h * w)) / (2 * h) - (_h(dg) * w).sum()) < 1e-6 + (
        (bd["dgamma"] + U * np.abs(_h(dg))) * np.abs(w)).sum()


def test_norm_and_dropout_refusals():
    from pdum_dsl_amd import kernels as K

    x = torch.randn((4, 8), device="cuda")
    f = K.layernorm_fwd(x)
    rng = torch.tensor([1, 2], device="cuda")
    for call, text in (
        (lambda: K.layernorm_fwd(x.double()), "f32, bf16 or f16"),
        (lambda: K.layernorm_fwd(x, torch.ones(7, device="cuda")), "vector of 8"),
        (lambda: K.layernorm_fwd(x, torch.ones(8, device="cuda", dtype=torch.bfloat16)), "element type"),
        (lambda: K.layernorm_fwd(x, eps=-1.0), "eps"),
        (lambda: K.layernorm_fwd(x, out=torch.empty(4, 9, device="cuda")), "x's shape"),
        (lambda: K.layernorm_fwd(x, out=torch.empty(1, 8, device="cuda").expand(4, 8)), "overlap"),
        (lambda: K.layernorm_fwd(x[:, :0]), "at least one column"),
        (lambda: K.layernorm_fwd(x.cpu()), "device tensors"),
        (lambda: K.layernorm_bwd(x, x[:3], f.mean, f.rstd), "dy must have"),
        (lambda: K.layernorm_bwd(x, x, f.mean[:3], f.rstd), "mean must be"),
        (lambda: K.layernorm_bwd(x, x, f.mean, f.rstd.double()), "rstd must be"),
        (lambda: K.layernorm_bwd(x, x, f.mean, f.rstd, dres=x.half()), "dres must have"),
        (lambda: K.dropout_fwd(x, 1.5, rng), "must lie in"),
        (lambda: K.dropout_fwd(x, float("nan"), rng), "must lie in"),
        (lambda: K.dropout_fwd(x, 0.1, rng, site=-1), "site"),
        (lambda: K.dropout_fwd(x, 0.1, rng.int()), "int64 device tensor"),
        (lambda: K.dropout_fwd(x, 0.1, torch.tensor([1, 2])), "device tensors"),
        (lambda: K.dropout_fwd(x, 0.1, rng, residual=x[:2]), "residual must"),
        (lambda: K.dropout_bwd(x.double(), 0.1, rng), "f32, bf16 or f16"),
    ):
        with pytest.raises(ValueError, match=text):
            call()


# --------------------------------------------------------------------- dropout


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,p", [((1, 1), 0.5), ((3, 7), 0.1), ((64, 768), 0.1), ((5, 8), 0.9), ((129, 1021), 0.25),
                                     ((2, 3, 40), 0.5), ((100,), 0.3), ((4, 64), 0.0), ((4, 64), 1.0), ((4, 64), 2.0**-17)])
def test_dropout_forward_and_backward(shape, p, dtype):
    """The mask is the oracle's exactly; a survivor is one multiplication (and
    one addition of the residual) and one rounding from its value."""
    from pdum_dsl_amd import kernels as K

    gen = np.random.default_rng(len(shape) * 100 + shape[-1])
    x, r, dy = (_draw(gen, shape, dtype) for _ in range(3))
    seed, step, site = 0x1234567890ABCDEF, (7 << 32) + 41, 0xFFFFFFFE
    rng = torch.tensor([seed, step], device="cuda")
    y = K.dropout_fwd(x, p, rng, site=site)
    yr = K.dropout_fwd(x, p, rng, site=site, residual=r)
    dx = K.dropout_bwd(dy, p, rng, site=site)
    torch.cuda.synchronize()
    for got, want, extra in ((y, cf.dropout(_h(x), p, seed, step, site), 0.0),
                             (yr, cf.dropout(_h(x), p, seed, step, site, _h(r)), 1.0),
                             (dx, cf.dropout(_h(dy), p, seed, step, site), 0.0)):
        kept = cf.dropout(np.abs(_h(x)) + np.abs(_h(dy)), p, seed, step, site)
        _within(got, want, 2 * U * kept + extra * U * np.abs(want), dtype, "dropout")
    if p < 1.0:
        assert np.array_equal(_h(y) != 0, cf.dropout(np.ones(shape), p, seed, step, site) * _h(x) != 0)


def test_dropout_rate_and_independence_of_layout_and_type():
    from pdum_dsl_amd import kernels as K

    rng = torch.tensor([99, 5], device="cuda")
    x = torch.ones((1000, 1003), device="cuda")
    y = K.dropout_fwd(x, 0.1, rng)
    n, p = x.numel(), 6554 / 65536
    kept = int((y != 0).sum())
    assert abs(kept - n * (1 - p)) < 6 * (n * p * (1 - p)) ** 0.5  # six standard deviations
    assert torch.equal(K.dropout_fwd(x.bfloat16(), 0.1, rng) != 0, y != 0)
    wide = torch.ones((1000, 1011), device="cuda")
    assert torch.equal(K.dropout_fwd(wide[:, 3:1006], 0.1, rng), y)
    for other in (K.dropout_fwd(x, 0.1, rng, site=1), K.dropout_fwd(x, 0.1, rng + torch.tensor([0, 1], device="cuda")),
                  K.dropout_fwd(x, 0.1, rng + torch.tensor([1, 0], device="cuda"))):
        both = int(((other != 0) & (y != 0)).sum())
        assert abs(both - n * (1 - p) ** 2) < 6 * (n * p) ** 0.5  # independent of the first
    z = x.clone()
    assert K.dropout_fwd(z, 0.1, rng, out=z) is z and torch.equal(z, y)


def test_dropped_elements_count_for_nothing():
    from pdum_dsl_amd import kernels as K

    rng = torch.tensor([3, 0], device="cuda")
    keep = K.dropout_fwd(torch.ones((50, 77), device="cuda"), 0.5, rng) != 0
    for bad in (float("nan"), float("inf")):
        x = torch.where(keep, torch.ones_like(keep, dtype=torch.float32), torch.full_like(keep, bad, dtype=torch.float32))
        assert torch.equal(K.dropout_fwd(x, 0.5, rng), 2.0 * keep)
        r = torch.randn((50, 77), device="cuda")
        assert torch.equal(K.dropout_fwd(x, 0.5, rng, residual=r), 2.0 * keep + r)


def test_a_captured_dropout_draws_the_masks_of_its_steps():
    """Forward and backward in one graph, the step moved on between replays:
    each replay equals the eager call at that step."""
    from pdum_dsl_amd import kernels as K

    x, dy = torch.randn((64, 500), device="cuda"), torch.randn((64, 500), device="cuda")
    rng = torch.tensor([11, 0], device="cuda")
    K.dropout_fwd(x, 0.2, rng)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dx = K.dropout_fwd(x, 0.2, rng, site=3), K.dropout_bwd(dy, 0.2, rng, site=3)
    seen = []
    for step in range(4):
        rng[1] = step
        x.copy_(torch.randn_like(x))
        want = K.dropout_fwd(x, 0.2, rng, site=3), K.dropout_bwd(dy, 0.2, rng, site=3)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and torch.equal(dx, want[1])
        seen.append(dx.clone())
    assert not any(torch.equal(seen[0], s) for s in seen[1:])


def test_a_captured_layernorm_step_replays():
    from pdum_dsl_amd import kernels as K

    x, dy = (torch.randn((300, 777), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    g = torch.randn(777, device="cuda", dtype=torch.bfloat16)

    def step():
        f = K.layernorm_fwd(x, g, g)
        return (f.y, f.mean, f.rstd) + K.layernorm_bwd(x, dy, f.mean, f.rstd, g, dres=dy)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        x.copy_(torch.randn((300, 777), device="cuda"))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_norm_and_dropout_on_a_side_stream():
    from pdum_dsl_amd import kernels as K

    x = torch.randn((500, 768), device="cuda")
    rng = torch.tensor([1, 2], device="cuda")
    want = K.layernorm_fwd(x).y, K.dropout_fwd(x, 0.1, rng)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = K.layernorm_fwd(x).y, K.dropout_fwd(x, 0.1, rng)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
