"""The paged-cache operators on the GPU where a program's calls differ from
the plain ones: drawn batches of any shape, many sequences, shared pages, pools
past 32-bit offsets and just short of them, lengths past the table, workspaces
full of NaN, captured prompts, tensors of another device."""

import ctypes as C

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


def _run(K, rng, dtype, bits, lengths, new, hq, hkv, d, pr, window=None, sinks=0, pad=0, scale=None, every=1, what=""):
    table, starts, lens, rows, pages = batch(rng, lengths, new, pr, pad=pad)
    cache, pk, pv = _pools(rng, K, dtype, bits, pages, hkv, pr, d)
    q = torch.as_tensor(rng.standard_normal((rows, hq, d))).to(DT[dtype]).cuda()
    o, lse = K.paged_attention(q, cache, *_ints(table, starts, lens), window=window, sinks=sinks, scale=scale)
    sc = d**-0.5 if scale is None else scale
    want = op.attention(_host(q), pk, pv, table, starts, lens, scale=sc, window=window, sinks=sinks, every=every)
    check_attention(_host(o), _host(lse), want, dtype, d, what)


@pytest.mark.parametrize("seed", range(24))
def test_drawn_batches(K, seed):
    rng = np.random.default_rng(1000 + seed)
    hkv = int(rng.choice([1, 2, 3, 5, 8]))
    hq = hkv * int(rng.choice([1, 2, 3, 4, 7, 16]))
    d, pr = int(rng.choice([64, 128])), int(rng.choice([16, 32, 128]))
    seqs = int(rng.integers(1, 7))
    lengths = [int(n) for n in np.exp(rng.uniform(0, np.log(900), seqs))]
    most = int(np.exp(rng.uniform(0, np.log(300))))
    new = [int(min(n, rng.integers(0, most + 1))) for n in lengths]
    window = None if rng.random() < 0.4 else int(np.exp(rng.uniform(0, np.log(300))))
    sinks = int(rng.choice([0, 0, 1, 4, 40, 200]))
    case = (str(rng.choice(["bf16", "f16"])), int(rng.choice([16, 4])), lengths, new, hq, hkv, d, pr, window, sinks,
            int(rng.choice([0, 0, 5, 140])))
    print(case, flush=True)
    if sum(new) + case[-1] == 0:
        new[0] = 1
    _run(K, rng, *case, scale=float(rng.choice([d**-0.5, 0.3])), every=max(1, max(new) // 25), what=str(case))


@pytest.mark.parametrize("bits", [16, 4])
def test_many_sequences(K, bits):
    """More than one sequence a thread of the decode kernel, some without rows, some without tokens."""
    rng = np.random.default_rng(21)
    lengths = [int(n) for n in rng.integers(0, 60, 700)]
    new = [int(n > 0 and rng.random() < 0.9) for n in lengths]
    lengths[613], new[613] = 3000, 1
    _run(K, rng, "bf16", bits, lengths, new, 4, 2, 64, 16, what="many")


@pytest.mark.parametrize("hq,hkv", [(16, 1), (3, 1)])
def test_one_long_sequence_over_every_workgroup(K, hq, hkv):
    _run(K, np.random.default_rng(22), "f16", 16, [40000], [1], hq, hkv, 64, 64, what="long")
    _run(K, np.random.default_rng(23), "bf16", 4, [40000], [2], hq, hkv, 64, 64, 9000, 5, what="long window")


@pytest.mark.parametrize("new", [[1, 1, 1], [30, 2, 17]])
def test_sequences_that_share_pages(K, new):
    """One prefix in three tables, twice in one of them."""
    rng = np.random.default_rng(24)
    pr, d, hq, hkv = 16, 64, 4, 2
    lengths = [60, 50, 90]
    cache, pk, pv = _pools(rng, K, "bf16", 16, 9, hkv, pr, d)
    table = np.array([[3, 1, 4, 0, 0, 0], [3, 1, 5, 2, 0, 0], [3, 1, 3, 1, 6, 7]], dtype=np.int32)
    starts = np.concatenate([[0], np.cumsum(new)])
    q = torch.as_tensor(rng.standard_normal((starts[-1], hq, d))).bfloat16().cuda()
    o, lse = K.paged_attention(q, cache, *_ints(table, starts, lengths))
    want = op.attention(_host(q), pk, pv, table, starts, lengths, scale=d**-0.5)
    check_attention(_host(o), _host(lse), want, "bf16", d, "shared")


@pytest.mark.parametrize("new", [[1, 1], [3, 70]])
def test_lengths_past_the_table(K, new):
    """Tokens that the table has no entry for are not seen; positions count on all the same."""
    rng = np.random.default_rng(25)
    pr, d, hq, hkv = 16, 64, 8, 2
    cache, pk, pv = _pools(rng, K, "bf16", 16, 6, hkv, pr, d)
    table = np.array([[0, 1, 2], [3, 4, 5]], dtype=np.int32)
    starts = np.concatenate([[0], np.cumsum(new)])
    q = torch.as_tensor(rng.standard_normal((starts[-1], hq, d))).bfloat16().cuda()
    for lengths, window, sinks in (([100, 75], None, 0), ([100, 75], 60, 3), ([2**31 - 1, 75], 60, 3), ([-5, 48], None, 0)):
        o, lse = K.paged_attention(q, cache, *_ints(table, starts, lengths), window=window, sinks=sinks)
        want = op.attention(_host(q), pk, pv, table, starts, [min(n, 1 << 20) for n in lengths], scale=d**-0.5, window=window,
                            sinks=sinks) if max(lengths) < 1000 else None
        if want is None:  # far past the table: the first sequence sees its first tokens alone
            near = op.attention(_host(q), pk, pv, table, starts, [5000, 75], scale=d**-0.5, window=window, sinks=sinks)
            want = near
        check_attention(_host(o), _host(lse), want, "bf16", d, str(lengths))


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("span", [0x7FFF0000 - 1, 0x7FFF0000, (1 << 32) + (1 << 20)])
def test_pools_about_the_reach_of_one_resource(K, bits, span):
    """The last page lies as far as one buffer resource reaches, right past it, and past 32 bits."""
    pr, d, hkv, hq = 16, 64, 1, 4
    unit = 2 if bits == 16 else 1
    row = d if bits == 16 else d // 2
    apart = (span // unit - pr * row) // 4 // 16 * 16  # four page distances and a page reach `span`
    rng = np.random.default_rng(26)
    kind = torch.bfloat16 if bits == 16 else torch.uint8
    k, v = (torch.zeros(apart * 4 + pr * row, dtype=kind, device="cuda").as_strided((5, hkv, pr, row), (apart, pr * row, row, 1))
            for _ in range(2))
    scales = [None, None] if bits == 16 else [torch.zeros((5, hkv, pr, d // 32), dtype=torch.uint8, device="cuda") for _ in range(2)]
    cache = K.PagedCache(k, v, *scales, torch.bfloat16)
    table = np.array([[4, 0, 3, 1, 2]], dtype=np.int32)
    lens = [77]
    x = torch.as_tensor(rng.standard_normal((77, hkv, d))).bfloat16().cuda()
    K.paged_append(x, x, cache, *_ints(table, [0, 77], lens))
    kk, vv = K.paged_rows(cache, *_ints(table, [0, 77], lens), 77)
    hk, hv = np.zeros((5, hkv, pr, d)), np.zeros((5, hkv, pr, d))
    for r in range(77):
        p, at = op.place(table, 0, r, pr, 5)
        hk[p, :, at], hv[p, :, at] = _host(kk[r]), _host(vv[r])
    if bits == 16:
        assert torch.equal(kk, x)
    for new in (1, 40, 77):
        q = torch.as_tensor(rng.standard_normal((new, hq, d))).bfloat16().cuda()
        o, lse = K.paged_attention(q, cache, *_ints(table, [0, new], lens), window=30, sinks=2)
        want = op.attention(_host(q), hk, hv, table, [0, new], lens, scale=d**-0.5, window=30, sinks=2)
        check_attention(_host(o), _host(lse), want, "bf16", d, f"{new} rows")


def test_a_row_that_is_not_a_number_spoils_itself_alone(K):
    for new in ([1, 2], [40, 3]):
        rng = np.random.default_rng(27)
        pr, d, hq, hkv = 16, 64, 8, 2
        table, starts, lens, rows, pages = batch(rng, [80, 50], new, pr)
        cache, pk, pv = _pools(rng, K, "bf16", 16, pages, hkv, pr, d)
        q = torch.as_tensor(rng.standard_normal((rows, hq, d))).bfloat16().cuda()
        want = op.attention(_host(q), pk, pv, table, starts, lens, scale=d**-0.5)
        q[1, 3, 7] = float("nan")
        o, lse = K.paged_attention(q, cache, *_ints(table, starts, lens))
        assert torch.isnan(o[1, 3]).all() and torch.isnan(lse[1, 3])
        o, lse = _host(o), _host(lse)
        o[1, 3], lse[1, 3] = want[0][1, 3], want[1][1, 3]
        check_attention(o, lse, want, "bf16", d, "a NaN in q")


def test_scores_of_minus_infinity_weigh_nothing(K):
    """Keys whose scores are -inf: left out of the softmax; rows with no other score see nothing."""
    rng = np.random.default_rng(28)
    pr, d, hq, hkv = 16, 64, 4, 2
    for new in ([1, 1], [60, 1]):
        table, starts, lens, rows, pages = batch(rng, [70, 33], new, pr)
        cache, pk, pv = _pools(rng, K, "bf16", 16, pages, hkv, pr, d)
        q = torch.as_tensor(np.abs(rng.standard_normal((rows, hq, d)))).bfloat16().cuda()
        for i, n in enumerate(lens):
            for s in range(n):
                if i == 1 or s % 3 == 0:
                    cache.k[table[i, s // pr], :, s % pr, 0] = -float("inf")
        o, lse = K.paged_attention(q, cache, *_ints(table, starts, lens))
        want = op.attention(_host(q), _host(cache.k), pv, table, starts, lens, scale=d**-0.5)
        assert (_host(o)[starts[1] :] == 0).all() and np.isneginf(_host(lse)[starts[1] :]).all()
        full = ~np.isneginf(want[1])
        S = np.where(np.isfinite(want[3]), want[3], 0)
        for r in range(starts[1]):  # the bound's largest score, without the infinite ones
            for h in range(hq):
                keys = [s for s in range(lens[0] - new[0] + r + 1) if s % 3]
                kk = np.array([_host(cache.k[table[0, s // pr], h // 2, s % pr]) for s in keys])
                S[r, h] = d**-0.5 * (np.abs(kk) @ np.abs(_host(q[r, h]))).max() if keys else 0.0
        want = (want[0], want[1], want[2], S, want[4], np.where(full, want[5], 0))
        check_attention(_host(o), _host(lse), want, "bf16", d, f"-inf scores {new}")


@pytest.mark.parametrize("bits,lengths,new", [(16, [3000, 20, 700], [1, 1, 1]), (4, [3000, 20], [2, 1]), (16, [6000], [130]),
                                              (4, [6000, 90], [70, 90])])
def test_workspaces_full_of_nan(K, bits, lengths, new):
    """No state is read that the call has not written; states and result repeat bit for bit."""
    from pdum_dsl_amd import _lib

    rng = np.random.default_rng(29)
    pr, d, hq, hkv = 16, 128, 8, 2
    table, starts, lens, rows, pages = batch(rng, lengths, new, pr, pad=3)
    cache, pk, pv = _pools(rng, K, "bf16", bits, pages, hkv, pr, d)
    q = torch.as_tensor(rng.standard_normal((rows, hq, d))).bfloat16().cuda()
    t = _ints(table, starts, lens)
    b = _lib.PagedBatch(t[0].data_ptr(), t[1].data_ptr(), t[2].data_ptr(), len(lens), rows, table.shape[1], table.shape[1])
    need = _lib.lib().pdh_paged_attention_workspace(C.byref(cache.c), C.byref(b), hq, 1 << 40, 0)
    assert need
    outs = []
    for fill in (float("nan"), 0.0, 1e30):
        ws = torch.full((need // 4,), fill, device="cuda")
        o, lse = torch.full_like(q, 9.0), torch.full((rows, hq), 9.0, device="cuda")
        _lib.call("pdh_paged_attention", q.data_ptr(), o.data_ptr(), lse.data_ptr(), hq, hq * d, d, hq * d, d, C.byref(cache.c),
                  C.byref(b), 1 << 40, 0, d**-0.5, 1, ws.data_ptr(), need, K._stream())
        outs.append((o, lse))
    for o, lse in outs[1:]:
        assert torch.equal(o, outs[0][0]) and torch.equal(lse, outs[0][1])
    want = op.attention(_host(q), pk, pv, table, starts, lens, scale=d**-0.5, every=9)
    check_attention(_host(outs[0][0]), _host(outs[0][1]), want, "bf16", d, "workspace")
    with pytest.raises(_lib.PdhError, match="workspace"):
        _lib.call("pdh_paged_attention", q.data_ptr(), o.data_ptr(), lse.data_ptr(), hq, hq * d, d, hq * d, d, C.byref(cache.c),
                  C.byref(b), 1 << 40, 0, d**-0.5, 1, ws.data_ptr(), need - 4, K._stream())


@pytest.mark.parametrize("new", [[200, 100], [1, 90]])
def test_captured_prompts_follow_their_inputs(K, new):
    """Pieces of prompts and a split grid as a graph, an eager call between the replays."""
    rng = np.random.default_rng(30)
    pr, d, hq, hkv = 16, 64, 4, 2
    table, starts, lens, rows, pages = batch(rng, [6000, 900], new, pr, width=400)
    cache, *_ = _pools(rng, K, "bf16", 16, pages, hkv, pr, d)
    q = torch.zeros((rows, hq, d), dtype=torch.bfloat16, device="cuda")
    t = _ints(table, starts, lens)
    step = lambda: K.paged_attention(q, cache, *t, window=5000, sinks=3)  # noqa: E731
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = step()
    for n in range(3):
        q.copy_(torch.as_tensor(rng.standard_normal(tuple(q.shape))).bfloat16())
        t[1].copy_(torch.tensor([0, new[0] - n, rows - 2 * n], dtype=torch.int32))  # some rows of no sequence
        t[2].copy_(torch.tensor([6000 - 700 * n, 900 - n], dtype=torch.int32))
        eo, el = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, eo) and torch.equal(lse, el), n


def test_a_window_past_everything_is_none(K):
    case = dict(dtype="bf16", bits=16, lengths=[200, 90], new=[100, 1], hq=4, hkv=2, d=64, pr=16)
    outs = []
    for window in (None, 200, 1 << 30, 1 << 62):
        rng = np.random.default_rng(31)
        table, starts, lens, rows, pages = batch(rng, case["lengths"], case["new"], 16)
        cache, *_ = _pools(rng, K, "bf16", 16, pages, 2, 16, 64)
        q = torch.as_tensor(rng.standard_normal((rows, 4, 64))).bfloat16().cuda()
        outs.append(K.paged_attention(q, cache, *_ints(table, starts, lens), window=window, sinks=1 << 40 if window else 0)[0])
    for o in outs[1:]:
        assert torch.equal(o, outs[0])


def test_tensors_of_another_device_are_refused(K, monkeypatch):
    cache = K.paged_cache(2, 2, 16, 64)
    cache.c  # described while its device is the current one
    t = _ints([[0]], [0, 1], [1])
    x = torch.zeros((1, 2, 64), dtype=torch.bfloat16, device="cuda")
    for bad in (dict(q=x.cpu()), dict(q=x.float()), dict(q=x, out=x.half()), dict(q=x, rotary=torch.zeros(4, 64)), dict(out=x)):
        with pytest.raises(ValueError):
            K.paged_append(x, x, cache, *t, **bad)
    for bad in (x.cpu(), x.float(), x[:, :1], x[0], x[:, :, :32]):
        with pytest.raises(ValueError):
            K.paged_attention(bad, cache, *t)
    with pytest.raises(ValueError, match="overlap"):
        K.paged_attention(x.expand(3, 2, 64), cache, *t, out=x.expand(3, 2, 64))
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1)
    for call in (lambda: K.paged_append(x, x, cache, *t), lambda: K.paged_rows(cache, *t, 1),
                 lambda: K.paged_attention(x, cache, *t)):
        with pytest.raises(ValueError, match="current device"):
            call()


@pytest.mark.parametrize("new", [1, 3, 130])
def test_an_infinite_value_is_its_rows_sum(K, new):
    """A value of +inf that a row sees: +inf in that feature, whatever parts the row's keys were cut into; nothing elsewhere."""
    rng = np.random.default_rng(31)
    pr, d, hq, hkv, n, key = 16, 64, 8, 2, 6000, 3
    table, starts, lens, rows, pages = batch(rng, [n], [new], pr)
    cache, pk, pv = _pools(rng, K, "bf16", 16, pages, hkv, pr, d)
    q = torch.as_tensor(rng.standard_normal((rows, hq, d))).bfloat16().cuda()
    want = op.attention(_host(q), pk, pv, table, starts, lens, scale=d**-0.5, every=max(1, new // 25))
    cache.v[table[0, 0], :, key, 5] = float("inf")
    o, lse = K.paged_attention(q, cache, *_ints(table, starts, lens))
    assert torch.isposinf(o[:, :, 5]).all()
    o = _host(o)
    o[:, :, 5] = want[0][:, :, 5]
    check_attention(o, _host(lse), want, "bf16", d, f"{new} rows")


@pytest.mark.parametrize("lengths,new", [([700, 90, 5], [1, 1, 1]), ([700, 90], [3, 2]), ([300, 200], [300, 40]), ([6000], [130])])
def test_attention_in_the_place_of_q(K, lengths, new):
    rng = np.random.default_rng(32)
    pr, d, hq, hkv = 16, 64, 8, 2
    table, starts, lens, rows, pages = batch(rng, lengths, new, pr, pad=3)
    cache, _, _ = _pools(rng, K, "bf16", 16, pages, hkv, pr, d)
    qkv = torch.as_tensor(rng.standard_normal((rows, hq + 2 * hkv, d))).bfloat16().cuda()
    q, held = qkv[:, :hq], qkv.clone()
    want, lse = K.paged_attention(q, cache, *_ints(table, starts, lens))
    got, lse2 = K.paged_attention(q, cache, *_ints(table, starts, lens), out=q)
    live = rows - 3
    assert got is q and torch.equal(q[:live], want[:live])
    assert torch.equal(lse, lse2) and torch.isneginf(lse[live:]).all()
    assert torch.equal(q[live:], held[live:, :hq]) and torch.equal(qkv[:, hq:], held[:, hq:])
    with pytest.raises(ValueError, match="q's strides"):
        K.paged_attention(q, cache, *_ints(table, starts, lens), out=q.as_strided((rows, hq, d), (hq * d, d, 1)))


def test_a_rotary_table_of_no_positions_has_room_for_no_token(K):
    cache = K.paged_cache(2, 2, 16, 64)
    x = torch.ones((3, 4, 64), dtype=torch.bfloat16, device="cuda")
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = K.paged_append(x[:, :2], x[:, 2:], cache, *_ints([[0]], [0, 3], [3]), q=x, rotary=K.rotary_table(0, 32), bad=bad)
    assert (got == 0).all() and (cache.k == 0).all() and (cache.v == 0).all() and int(bad) == 3


def test_no_rows_to_append(K):
    cache = K.paged_cache(2, 2, 16, 64)
    x = torch.empty((0, 8, 64), dtype=torch.bfloat16, device="cuda")
    got = K.paged_append(x[:, 4:6], x[:, 6:], cache, *_ints([[0]], [0, 0], [7]), q=x[:, :4], rotary=K.rotary_table(9, 64))
    assert got.shape == (0, 4, 64) and (cache.k == 0).all()


@pytest.mark.parametrize("dtype,bits,hq,hkv,d,rotated,pairs", [
    ("bf16", 16, 32, 8, 128, 128, False), ("f16", 4, 32, 8, 128, 64, True), ("bf16", 4, 13, 13, 64, 64, False),
    ("f16", 16, 7, 3, 64, 16, True), ("bf16", 16, 0, 40, 128, 0, False),
])
def test_a_large_batch_is_its_small_ones(K, dtype, bits, hq, hkv, d, rotated, pairs):
    """Rows enough for several chunks a thread (over 2^18 of 8 features in all): the bits of the same rows appended a few at a time."""
    rng = np.random.default_rng(33)
    lengths, pr = [3001, 40, 1500, 0, 777], 32
    new = [int(min(n, m)) for n, m in zip(lengths, [2900, 40, 1499, 0, 500])]
    table, starts, lens, rows, pages = batch(rng, lengths, new, pr, pad=17)
    assert rows * (hq + 2 * hkv) * (d // 8) > 1 << 18
    table[2, 5] = pages  # a page outside the pool: its tokens are dropped
    caches = [K.paged_cache(pages, hkv, pr, d, DT[dtype], bits=bits) for _ in range(2)]
    x = torch.as_tensor(rng.standard_normal((rows, max(hq, 1) + 2 * hkv, d))).to(DT[dtype]).cuda()
    q, k, v = (x[:, :hq] if hq else None), x[:, -2 * hkv : -hkv], x[:, -hkv:]
    rot = K.rotary_table(3000, rotated) if rotated else None  # the first sequence's last token lies past it
    bad = torch.zeros(2, dtype=torch.int32, device="cuda")
    got = K.paged_append(k, v, caches[0], *_ints(table, starts, lens), q=q, rotary=rot, interleaved=pairs, bad=bad[:1])
    for i in range(len(lens)):
        for r in range(starts[i], starts[i + 1], 150):
            n = min(150, starts[i + 1] - r)
            t = _ints(table[i : i + 1], [0, n], [lens[i] - (starts[i + 1] - r) + n])
            part = K.paged_append(k[r : r + n], v[r : r + n], caches[1], *t, q=q[r : r + n] if hq else None, rotary=rot,
                                  interleaved=pairs, bad=bad[1:])
            assert not hq or torch.equal(part, got[r : r + n])
    assert not hq or (got[starts[-1] :] == 0).all()
    assert int(bad[0]) == int(bad[1]) == 32 + bool(rotated)
    for a, b in ((getattr(c, n) for c in caches) for n in ("k", "v", "k_scale", "v_scale") if bits == 4 or len(n) == 1):
        assert torch.equal(a, b)
    if hq:  # in q's place
        turned = x.clone()
        at = turned[:, :hq]
        K.paged_append(k, v, caches[1], *_ints(table, starts, lens), q=at, rotary=rot, interleaved=pairs, out=at)
        assert torch.equal(at[: starts[-1]], got[: starts[-1]]) and torch.equal(turned[starts[-1] :], x[starts[-1] :])
