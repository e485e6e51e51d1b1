"""The training operators over rows far apart and rows as wide as a call takes:
as the contiguous call, bit for bit, or within the closed forms' bounds."""

import numpy as np
import pytest

from tests.test_gpu_linear_xent import DTYPES, _check, _draw

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def _apart(a, stride):
    """a's rows `stride` elements apart, in memory full of NaN."""
    rows, cols = a.shape
    big = torch.full(((rows - 1) * stride + cols + 8,), float("nan"), dtype=a.dtype, device="cuda")
    view = big.as_strided((rows, cols), (stride, 1))
    view.copy_(a)
    return view


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("far", ["x", "w", "both"])
@pytest.mark.parametrize("stride", [1 << 21, (1 << 21) + 8])
def test_a_head_whose_rows_lie_far_apart(stride, far, dtype):
    """2^21 elements are the most that rows are read in place at; past it they are copied."""
    from pdum_dsl_amd import kernels as K

    rng = np.random.default_rng(stride % 97)
    n, d, v = 140, 72, 270
    x, w = _draw(rng, (n, d), dtype), _draw(rng, (v, d), dtype, 0.2)
    t = torch.as_tensor(rng.integers(0, v, n)).cuda()
    dloss = torch.rand(n, device="cuda")
    f = K.linear_cross_entropy(x, w, t)
    want = (f.loss, f.lse) + K.linear_cross_entropy_bwd(x, w, t, f.lse, dloss)
    x, w = (_apart(x, stride) if far != "w" else x), (_apart(w, stride) if far != "x" else w)
    f = K.linear_cross_entropy(x, w, t)
    got = (f.loss, f.lse) + K.linear_cross_entropy_bwd(x, w, t, f.lse, dloss)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,d,v", [(3, 1 << 18, 50), (130, (1 << 18) - 1, 5)])
def test_a_head_as_wide_as_a_call_takes(n, d, v, dtype):
    from pdum_dsl_amd import kernels as K

    rng = np.random.default_rng(n)
    x, w = _draw(rng, (n, d), dtype), _draw(rng, (v, d), dtype, 2.0 * d**-0.5)
    t = torch.as_tensor(rng.integers(0, v, n)).cuda()
    dloss = torch.as_tensor(rng.standard_normal(n) / n, dtype=torch.float32).cuda()
    f = K.linear_cross_entropy(x, w, t)
    g = K.linear_cross_entropy_bwd(x, w, t, f.lse, dloss)
    torch.cuda.synchronize()
    _check(x, w, t, dloss, f, g, dtype)


@pytest.mark.parametrize("cols", [3, 100, 1030, 20001])
def test_norm_and_dropout_over_rows_past_32_bits(cols):
    """Two rows more than 2^31 elements apart, in and out."""
    from pdum_dsl_amd import kernels as K

    rng = np.random.default_rng(cols)
    x, dy = (_draw(rng, (2, cols), torch.bfloat16) for _ in range(2))
    g, r = _draw(rng, cols, torch.bfloat16), torch.tensor([5, 6], device="cuda")
    stride = (1 << 31) + 24
    far = torch.zeros(stride + cols, dtype=torch.bfloat16, device="cuda").as_strided((2, cols), (stride, 1))
    want = K.layernorm_fwd(x, g, g)
    grads = K.layernorm_bwd(x, dy, want.mean, want.rstd, g, dres=x)
    drop = K.dropout_fwd(x, 0.3, r, residual=dy)
    far.copy_(x)
    got = K.layernorm_bwd(far, dy, want.mean, want.rstd, g, dres=far)
    assert all(torch.equal(a, b) for a, b in zip(got, grads))
    assert torch.equal(K.dropout_fwd(far, 0.3, r, residual=dy, out=far), drop)
    far.copy_(x)
    f = K.layernorm_fwd(far, g, g, out=far)
    assert all(torch.equal(a, b) for a, b in ((f.y, want.y), (f.mean, want.mean), (f.rstd, want.rstd)))
