"""The paged-cache operators on the GPU where a table, starts or lengths are not what a call means: pages that are missing,
rows that no sequence owns, sequences that go on behind the call's rows, lengths past every table."""

import numpy as np
import pytest

from tests.paged_cases import batch, check_attention, op
from tests.test_gpu_paged import DT, _host, _ints, _pools

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def K():
    from pdum_dsl_amd import kernels

    return kernels


@pytest.mark.parametrize("dtype,bits", [("bf16", 16), ("f16", 16), ("bf16", 4), ("f16", 4)])
@pytest.mark.parametrize("missing", [-1, 1 << 20])
@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("window", [None, 70])
def test_a_missing_page_is_not_another_ones(K, dtype, bits, missing, half, window):
    """Single tokens beside a piece, each without one page of the last 32 keys that it should see whole: neither the first
    page of the pool nor the last, which hold infinities and NaN and are nobody's, stand in for it."""
    rng = np.random.default_rng(40)
    pr, d, hq, hkv = 16, 64, 8, 2
    lengths, new = [40, 104, 33, 96, 200, 150], [1, 1, 1, 1, 1, 100]
    table, starts, lens, rows, pages = batch(rng, lengths, new, pr)
    cache, pk, pv = _pools(rng, K, dtype, bits, pages, hkv, pr, d)
    used = set(table[table >= 0].tolist())
    free = sorted(set(range(pages)) - used)[:2]
    swap = {0: free[0], pages - 1: free[1]}  # pages 0 and the last are to be nobody's
    swap = {a: b for a, b in swap.items() if a in used}
    table = np.vectorize(lambda p: swap.get(p, p))(table).astype(np.int32)
    for i, n in enumerate(lengths):
        table[i, 2 * ((n >> 5) - 1) + half] = missing
    for page in (0, pages - 1):
        assert page not in table
        if bits == 16:
            cache.k[page], cache.v[page] = float("nan"), float("inf")
            cache.v[page, :, ::2] = float("nan")
        else:
            cache.k_scale[page] = cache.v_scale[page] = 255
    q = torch.as_tensor(rng.standard_normal((rows, hq, d))).to(DT[dtype]).cuda()
    o, lse = K.paged_attention(q, cache, *_ints(table, starts, lens), window=window, sinks=2)
    want = op.attention(_host(q), pk, pv, table, starts, lens, scale=d**-0.5, window=window, sinks=2)
    check_attention(_host(o), _host(lse), want, dtype, d, f"missing {missing}, half {half}")
