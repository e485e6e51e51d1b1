"""The layer norm backward over a workspace full of NaN: no partial sum is added
that no workgroup wrote, and nothing is written past the workspace."""

import numpy as np
import pytest

from tests.test_gpu_norm_dropout import _draw

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(1, 768), (7, 100), (2050, 1023), (2049, 3), (63, 5), (513, 1500), (255, 5000), (257, 8192),
                                       (300, 9001), (65, 16401)])
def test_the_weights_sums_read_only_what_was_written(rows, cols, dtype):
    from pdum_dsl_amd import _lib
    from pdum_dsl_amd import kernels as K

    rng = np.random.default_rng(rows)
    x, dy, g = _draw(rng, (rows, cols), dtype), _draw(rng, (rows, cols), dtype), _draw(rng, cols, dtype)
    f = K.layernorm_fwd(x, g)
    code = K._DT[dtype]
    need = _lib.lib().pdh_layernorm_bwd_workspace(rows, cols, code)
    out = []
    for fill in (255, 0):
        ws = torch.full((need + 4096,), fill, dtype=torch.uint8, device="cuda")
        dx, dg, db = torch.empty_like(x), torch.empty_like(g), torch.empty_like(g)
        _lib.call("pdh_layernorm_bwd", x.data_ptr(), dy.data_ptr(), None, g.data_ptr(), f.mean.data_ptr(),
                  f.rstd.data_ptr(), dx.data_ptr(), dg.data_ptr(), db.data_ptr(), rows, cols, cols, cols, 0, cols, code,
                  ws.data_ptr(), need, K._stream())
        assert (ws[need:] == fill).all()
        out.append((dx, dg, db))
    for a, b, c in zip(*out, K.layernorm_bwd(x, dy, f.mean, f.rstd, g)):
        assert torch.isfinite(a).all() and torch.equal(a, b) and torch.equal(a, c)
