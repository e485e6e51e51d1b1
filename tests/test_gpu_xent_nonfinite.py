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
