"""The linear head's gradient where a weight or an entry of the head is not
finite: what is not finite spoils what the formulas give it and nothing else."""

import numpy as np
import pytest

from tests.test_gpu_linear_xent import DTYPES, _draw

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("scale", [1e-3, 100.0])
def test_one_weight_that_is_not_finite_spoils_its_own_token(dtype, bad, scale):
    """Under a loss scale one token's dloss overflowed: the other tokens' dx are,
    bit for bit, those of a finite weight there (no larger than the others')."""
    from pdum_dsl_amd import kernels as K

    rng = np.random.default_rng(21)
    n, d, v = 70, 96, 700
    x, w = _draw(rng, (n, d), dtype), _draw(rng, (v, d), dtype, 0.2)
    t = torch.as_tensor(rng.integers(0, v, n)).cuda()
    dloss = torch.as_tensor(scale * (rng.random(n) + 0.5), dtype=torch.float32).cuda()
    f = K.linear_cross_entropy(x, w, t)
    dloss[11] = scale / 4
    want, _ = K.linear_cross_entropy_bwd(x, w, t, f.lse, dloss)
    dloss[11] = bad
    dx, _ = K.linear_cross_entropy_bwd(x, w, t, f.lse, dloss)
    rest = torch.arange(n, device="cuda") != 11
    assert torch.isfinite(dx[rest]).all() and torch.equal(dx[rest], want[rest])
    assert not torch.isfinite(dx[11]).any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("n,d,v", [(90, 64, 700), (1100, 72, 333), (300, 256, 2049)])
def test_ignored_tokens_have_no_gradient_whatever_the_head_holds(n, d, v, bad, dtype):
    """An entry of w that is not finite: dx of ignored tokens is zero, and where no token is live so is dw."""
    from pdum_dsl_amd import kernels as K

    rng = np.random.default_rng(n)
    x, w = _draw(rng, (n, d), dtype), _draw(rng, (v, d), dtype, 0.2)
    w[v // 2, 3] = bad
    t = torch.as_tensor(rng.integers(0, v, n)).cuda()
    t[::3] = -100
    t[4] = v
    dead = (t < 0) | (t >= v)
    dloss = torch.full((n,), 1.0 / n, device="cuda")
    f = K.linear_cross_entropy(x, w, t)
    dx, _ = K.linear_cross_entropy_bwd(x, w, t, f.lse, dloss)
    assert not f.loss[dead].any() and not dx[dead].any() and not torch.isfinite(dx[~dead]).all()
    none = torch.full_like(t, -100)
    f = K.linear_cross_entropy(x, w, none)
    dx, dw = K.linear_cross_entropy_bwd(x, w, none, f.lse, dloss)
    assert not f.loss.any() and not dx.any() and not dw.any()


@pytest.mark.parametrize("dtype", DTYPES[1:])
def test_an_entry_of_logits_minus_infinity_leaves_dw_finite(dtype):
    """-inf in a feature that is positive in every token: the entry's probability is zero, and so is its row of dw,
    ignored tokens or not."""
    from pdum_dsl_amd import kernels as K

    rng = np.random.default_rng(8)
    n, d, v = 200, 64, 500
    x, w = _draw(rng, (n, d), dtype), _draw(rng, (v, d), dtype, 0.2)
    x[:, 3] = x[:, 3].abs() + 0.5
    t = torch.as_tensor(rng.integers(0, v - 1, n)).cuda()
    t[::4] = -100
    w[v - 1, 3] = -float("inf")
    dloss = torch.full((n,), 1.0 / n, device="cuda")
    f = K.linear_cross_entropy(x, w, t)
    _, dw = K.linear_cross_entropy_bwd(x, w, t, f.lse, dloss)
    assert torch.isfinite(f.loss).all() and torch.isfinite(dw).all() and not dw[v - 1].any() and dw[:-1].any(1).all()
