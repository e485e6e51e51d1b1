"""The linear head's loss over workspaces that hold NaN: nothing is summed that
no kernel wrote. Tolerances are tests/test_gpu_linear_xent.py's, whose M = 4 k /
16 roundings of a sum of k products also hold for a sum in parts: a part is 256
products at least, 64 of those roundings, and joining it adds one."""

import numpy as np
import pytest

from tests.test_gpu_linear_xent import _check, _draw

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _case(n, d, v, dtype, seed=0):
    rng = np.random.default_rng(seed + n + d + v)
    x, w = _draw(rng, (n, d), dtype), _draw(rng, (v, d), dtype, 2.0 * d**-0.5)
    ht = rng.integers(0, v, n)
    ht[1:][rng.random(n - 1) < 0.1] = -100
    dloss = torch.as_tensor(rng.standard_normal(n) / n, dtype=torch.float32).cuda()
    return x, w, torch.as_tensor(ht).cuda(), dloss


def _run(x, w, t, dloss, fill):
    """Loss, lse, dx and dw through the C entry points, their workspaces full of `fill`."""
    from pdum_dsl_amd import _lib
    from pdum_dsl_amd import kernels as K

    lib, code = _lib.lib(), K._DT[x.dtype]
    sizes = (x.shape[0], x.shape[1], w.shape[0], x.shape[1], x.shape[1])

    def space(backward):
        need = lib.pdh_linear_xent_workspace(x.data_ptr(), w.data_ptr(), *sizes, code, backward)
        return torch.full((need,), fill, dtype=torch.uint8, device="cuda"), need

    loss, lse = torch.empty_like(dloss), torch.empty_like(dloss)
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    ws, need = space(0)
    _lib.call("pdh_linear_xent_fwd", x.data_ptr(), w.data_ptr(), t.data_ptr(), loss.data_ptr(), lse.data_ptr(), *sizes,
              -100, code, None, ws.data_ptr(), need, K._stream())
    ws, need = space(1)
    _lib.call("pdh_linear_xent_bwd", x.data_ptr(), w.data_ptr(), t.data_ptr(), lse.data_ptr(), dloss.data_ptr(),
              dx.data_ptr(), dw.data_ptr(), *sizes, -100, code, ws.data_ptr(), need, K._stream())
    return loss, lse, dx, dw


@pytest.mark.parametrize("n,d,v,dtype", [
    (64, 1024, 16000, BF16), (1, 512, 16000, BF16), (300, 768, 8000, BF16), (300, 768, 8000, F16), (128, 512, 20000, F32),
    (1326, 128, 2113, F32), (1774, 128, 4462, BF16), (268, 448, 16923, F16),
])
def test_vocabularies_that_end_inside_a_slice_of_whole_tiles(n, d, v, dtype):
    """The last slice of dx's product would lie past the vocabulary if it were counted over whole tiles."""
    from pdum_dsl_amd import kernels as K

    x, w, t, dloss = _case(n, d, v, dtype)
    loss, lse, dx, dw = _run(x, w, t, dloss, 255)
    torch.cuda.synchronize()
    _check(x, w, t, dloss, K.LossOut(loss, lse), (dx, dw), dtype)


@pytest.mark.parametrize("n,d,v,dtype", [
    (100, 768, 5003, BF16), (1024, 768, 50257, F32), (8192, 768, 50257, BF16), (777, 1023, 5003, F16), (16, 768, 6657, BF16),
    (594, 1294, 2127, F32), (128, 1024, 30522, BF16), (3000, 200, 70001, F32), (4500, 8, 9, F16), (2000, 64, 12345, BF16),
    (1, 1, 1, F32), (257, 40, 2049, F16), (5000, 320, 300, BF16), (40, 4096, 32000, F16),
])
def test_results_do_not_depend_on_what_the_workspace_held(n, d, v, dtype):
    case = _case(n, d, v, dtype, 1)
    a, b = _run(*case, 255), _run(*case, 0)
    torch.cuda.synchronize()
    for p, q in zip(a, b):
        assert torch.isfinite(p).all() and torch.equal(p, q)
