"""The training operators past 32 bits: operands of more than 2^31 elements, the
largest numbers of tokens and entries, and calls that take several launches.
Rows that a short call can compute alone are compared bit for bit; the rest
with float64 formulas on the device, in chunks, under the bounds of
tests/test_gpu_linear_xent.py given the device's lse."""

import numpy as np
import pytest

from oracle import closed_forms as cf

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = 2.0**-24
BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def _memory():
    yield
    torch.cuda.empty_cache()


def _normal(gen, *shape, std=1.0):
    return torch.empty(shape, dtype=BF16, device="cuda").normal_(0.0, std, generator=gen)


def _m(k):  # a sum of k products by the matrix cores, as the module named above derives it
    return 6 * U * (4 * -(-k // 16)) ** 0.5


def _chunk(x, w, t, lse, g, lo):
    """dz of entries lo .. lo + len(w) - 1 for x's tokens, and its error's bound."""
    z = x @ w.T
    ep = _m(x.shape[1]) * (z.abs() + 4 * ((x**2) @ (w**2).T).sqrt()) + 4 * U * (z.abs() + lse.abs() + 1)
    p = torch.exp(z - lse)
    dz = p.clone()
    hit = (t >= lo) & (t < lo + w.shape[0])
    dz[hit.nonzero()[:, 0], t[hit] - lo] -= 1.0
    dz *= g
    return z, dz, 2.0**-8 * dz.abs() + g.abs() * (p * ep + 2 * U)


def _within(got, want, err, what):
    assert ((got.double() - want).abs() <= err + 2.0**-8 * (want.abs() + err)).all(), what


def test_as_many_entries_as_a_call_takes():
    """2^24 entries of a head of 2.3e9 elements, four pieces of 2^22: few tokens. lse joins 2048 strips in a lane: 6 u
    sqrt(2048 + 2 * 128) < 300 u beside a logit's error."""
    from pdum_dsl_amd import kernels as K

    gen = torch.Generator(device="cuda").manual_seed(1)
    n, d, v, step = 24, 136, 1 << 24, 1 << 19
    x, w = _normal(gen, n, d), _normal(gen, v, d, std=0.15)
    t = torch.randint(0, v, (n,), generator=gen, device="cuda")
    t[:3] = torch.tensor([v - 1, -100, (1 << 22) - 1], device="cuda")
    dloss = torch.rand(n, generator=gen, device="cuda") + 0.5
    f = K.linear_cross_entropy(x, w, t)
    dx, dw = K.linear_cross_entropy_bwd(x, w, t, f.lse, dloss)
    live = t >= 0
    hx, lse = x.double(), f.lse.double()[:, None]
    g = (dloss.double() * live)[:, None]
    wx, ex, qx = (torch.zeros((n, d), dtype=torch.float64, device="cuda") for _ in range(3))
    total, zt = torch.zeros(n, dtype=torch.float64, device="cuda"), torch.zeros(n, dtype=torch.float64, device="cuda")
    zmax = torch.zeros(n, dtype=torch.float64, device="cuda")
    for lo in range(0, v, step):
        wc = w[lo:lo + step].double()
        z, dz, e = _chunk(hx, wc, t, lse, g, lo)
        total += torch.exp(z - lse).sum(1)
        zmax = torch.maximum(zmax, z.abs().max(1).values)
        hit = (t >= lo) & (t < lo + step)
        zt[hit] = z[hit.nonzero()[:, 0], t[hit] - lo]
        wx += dz @ wc
        ex += e @ wc.abs()
        qx += (dz**2) @ (wc**2)
        want = dz.T @ hx
        _within(dw[lo:lo + step], want, e.T @ hx.abs() + _m(n) * (want.abs() + 4 * ((dz**2).T @ (hx**2)).sqrt()), lo)
    want = f.lse.double() + torch.log(total)
    size = (hx**2).sum(1).sqrt() * (w[:4096].double() ** 2).sum(1).max().sqrt()  # |z|'s terms: 4 sqrt of their squares' sum
    ez = _m(d) * (zmax + 4 * size)
    assert ((f.lse.double() - want).abs() <= ez + 4 * U * (zmax + want.abs()) + 300 * U).all()
    loss = torch.where(live, want - zt, torch.zeros_like(want))
    assert ((f.loss.double() - loss).abs() <= 2 * ez + 8 * U * (zmax + want.abs()) + 300 * U).all() and not dx[1].any()
    _within(dx, wx, ex + _m(v) * (wx.abs() + 4 * qx.sqrt()), "dx")


def test_as_many_tokens_as_a_call_takes():
    """2^24 tokens of 136 features, 2.3e9 elements, over a small vocabulary."""
    from pdum_dsl_amd import kernels as K

    gen = torch.Generator(device="cuda").manual_seed(2)
    n, d, v, step = 1 << 24, 136, 20, 1 << 20
    x, w = _normal(gen, n, d), _normal(gen, v, d, std=0.15)
    t = torch.randint(0, v, (n,), generator=gen, device="cuda")
    t[::5] = -100
    dloss = torch.rand(n, generator=gen, device="cuda")
    f = K.linear_cross_entropy(x, w, t)
    dx, dw = K.linear_cross_entropy_bwd(x, w, t, f.lse, dloss)
    hw = w.double()
    ww, ew, qw = (torch.zeros((v, d), dtype=torch.float64, device="cuda") for _ in range(3))
    for lo in range(0, n, step):
        at = slice(lo, lo + step)
        hx, lse, g = x[at].double(), f.lse[at].double()[:, None], (dloss[at].double() * (t[at] >= 0))[:, None]
        z, dz, e = _chunk(hx, hw, t[at], lse, g, 0)
        real = torch.logsumexp(z, 1)
        ez = _m(d) * (z.abs() + 4 * ((hx**2) @ (hw**2).T).sqrt())
        lim = ez.max(1).values + 4 * U * (z.abs().max(1).values + real.abs()) + 200 * U
        assert ((lse[:, 0] - real).abs() <= lim).all(), lo
        want = dz @ hw
        _within(dx[at], want, e @ hw.abs() + _m(v) * (want.abs() + 4 * ((dz**2) @ (hw**2)).sqrt()), lo)
        assert not dx[at][t[at] < 0].any() and not f.loss[at][t[at] < 0].any()
        ww += dz.T @ hx
        ew += e.T @ hx.abs()
        qw += (dz**2).T @ (hx**2)
    _within(dw, ww, ew + _m(n) * (ww.abs() + 4 * qw.sqrt()), "dw")


@pytest.mark.parametrize("rows,cols", [((1 << 21) + 9, 1032), ((1 << 20) + 3, 2049), ((1 << 21) + 9, 3)])
def test_layernorm_over_many_rows(rows, cols):
    """More than 2^31 elements, more rows than a forward's launch holds: the first and last rows are a short call's,
    the weights' gradients the formulas'. A lane adds rows / 256 values at most (rows / 64 / 4 in the narrow rows)
    and another 160: random signs, 6 sqrt of that many roundings of the largest partial sum."""
    from pdum_dsl_amd import kernels as K

    gen = torch.Generator(device="cuda").manual_seed(rows + cols)
    x, dy = _normal(gen, rows, cols), _normal(gen, rows, cols)
    gamma, beta = 1 + _normal(gen, cols, std=0.1), _normal(gen, cols, std=0.1)
    f = K.layernorm_fwd(x, gamma, beta)
    dx, dgamma, dbeta = K.layernorm_bwd(x, dy, f.mean, f.rstd, gamma, dres=dy)
    for at in (slice(0, 40), slice((1 << 20) - 20, (1 << 20) + 20), slice(rows - 40, rows)):
        h = K.layernorm_fwd(x[at], gamma, beta)
        want = (h.y, h.mean, h.rstd, K.layernorm_bwd(x[at], dy[at], h.mean, h.rstd, gamma, dres=dy[at])[0])
        assert all(torch.equal(a[at], b) for a, b in zip((f.y, f.mean, f.rstd, dx), want))
    sums = torch.zeros((4, cols), dtype=torch.float64, device="cuda")
    for lo in range(0, rows, 1 << 17):
        at = slice(lo, lo + (1 << 17))
        xc = x[at].double()
        xc -= xc.mean(1, keepdim=True)
        xh, d = xc / ((xc * xc).mean(1, keepdim=True) + 1e-5).sqrt(), dy[at].double()
        sums += torch.stack([(d * xh).sum(0), d.sum(0), ((d * xh) ** 2).sum(0), (d * d).sum(0)])
    m = 6 * U * (rows / 256 + 160) ** 0.5
    for got, want, sq in ((dgamma, sums[0], sums[2]), (dbeta, sums[1], sums[3])):
        _within(got, want, (m + 50 * U) * (want.abs() + 4 * sq.sqrt()), "weights")


def test_dropout_over_more_groups_than_a_launch():
    """2^31 + 8 rows of one column: the second launch goes on where the first one's positions end."""
    from pdum_dsl_amd import kernels as K

    rows, seed, step = (1 << 31) + 8, 0x1234567890ABCDEF, 77
    x = torch.full((rows, 1), 3.0, dtype=BF16, device="cuda")
    y = K.dropout_fwd(x, 0.25, torch.tensor([seed, step], device="cuda"), site=5)
    for lo in (0, 1 << 30, (1 << 31) - 40):
        keep = cf.philox_bits(seed, step, 5, 48, 1, row0=lo)[:, 0] >= 16384
        assert np.array_equal(y[lo:lo + 48, 0].float().cpu().numpy(), np.where(keep, 4.0, 0.0))
