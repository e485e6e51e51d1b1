"""The training operators together, as a step uses them: a tied embedding
gathered, a branch dropped out onto the residual stream, the norm, the head's
loss over the same table, and the way back to the table's gradient (the head's
plus the gather's scatter), against float64 autograd under the oracle's mask.

Tolerances: the repository's statement for whole chains, 1e-5 of scale for fp32
and 2e-2 of scale for 16-bit storage (every stored value rounds once; the
single operators are held to derived bounds in their own tests)."""

import pytest

from oracle import closed_forms as cf

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

P, EPS, SITE = 0.1, 1e-5, 3


def _inputs(n, d, v, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s, std=1.0: (std * torch.randn(s, generator=g, device="cuda")).to(dtype)  # noqa: E731
    ids = torch.randint(0, v, (n,), generator=g, device="cuda")
    t = torch.randint(0, v, (n,), generator=g, device="cuda")
    t[:: 7] = -100
    live = (t != -100).float()
    return dict(table=r(v, d, std=0.5), ids=ids, t=t, gamma=1 + r(d, std=0.1), beta=r(d, std=0.1), c=r(n, d, std=1e-3),
                dloss=live / live.sum(), rng=torch.tensor([seed, 11], device="cuda"))


def _step(K, s):
    """Loss and the gradients of the table, gamma and beta, of mean loss + sum(c h)."""
    x = K.take_rows(s["table"], s["ids"])
    h = K.dropout_fwd(torch.tanh(x), P, s["rng"], site=SITE, residual=x)
    f = K.layernorm_fwd(h, s["gamma"], s["beta"], EPS)
    o = K.linear_cross_entropy(f.y, s["table"], s["t"])
    dy, dhead = K.linear_cross_entropy_bwd(f.y, s["table"], s["t"], o.lse, s["dloss"])
    dh, dgamma, dbeta = K.layernorm_bwd(h, dy, f.mean, f.rstd, s["gamma"], dres=s["c"])
    dtanh = K.dropout_bwd(dh, P, s["rng"], site=SITE)
    dx = dh + dtanh * (1 - torch.tanh(x) ** 2)
    dtable = dhead + K.scatter_add_rows(dx, s["ids"], s["table"].shape[0])
    return o.loss, dtable, dgamma, dbeta


def _oracle(s):
    d = {k: v.double().detach() for k, v in s.items() if v.is_floating_point()}
    for k in ("table", "gamma", "beta"):
        d[k].requires_grad_()
    x = d["table"][s["ids"]]
    seed, step = s["rng"].tolist()
    ones = torch.ones(x.shape, device="cpu").double().numpy()
    keep = torch.as_tensor(cf.dropout(ones, P, seed, step, SITE), device="cuda")
    h = x + torch.tanh(x) * keep
    mu = h.mean(-1, keepdim=True)
    y = (h - mu) / torch.sqrt(((h - mu) ** 2).mean(-1, keepdim=True) + EPS) * d["gamma"] + d["beta"]
    z = y @ d["table"].T
    live = s["t"] != -100
    loss = torch.where(live, torch.logsumexp(z, 1) - z.gather(1, s["t"].clamp(min=0)[:, None])[:, 0], 0.0)
    ((loss * d["dloss"]).sum() + (h * d["c"]).sum()).backward()
    return loss.detach(), d["table"].grad, d["gamma"].grad, d["beta"].grad


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-5), (torch.bfloat16, 2e-2), (torch.float16, 2e-2)])
@pytest.mark.parametrize("n,d,v", [(130, 96, 501), (257, 264, 1000), (64, 61, 77)])
def test_a_training_step(n, d, v, dtype, tol):
    from pdum_dsl_amd import kernels as K

    s = _inputs(n, d, v, dtype, n + d)
    for got, want, what in zip(_step(K, s), _oracle(s), ("loss", "dtable", "dgamma", "dbeta")):
        err, scale = (got.double() - want).abs().max().item(), max(want.abs().max().item(), 1e-30)
        assert err <= tol * scale, f"{what}: {err:.3e} of {scale:.3e}"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_captured_step_draws_new_masks_and_repeats_the_eager_one(dtype):
    """The whole step in one graph; between replays the generator's step moves
    on, the ids change and an eager step runs. Two graphs of the same tensors
    replay in turn."""
    from pdum_dsl_amd import kernels as K

    s = _inputs(200, 128, 700, dtype, 5)
    for _ in range(2):
        _step(K, s)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _step(K, s)
        graphs.append((graph, out))
    losses = []
    for rep in range(4):
        s["rng"][1] += 1
        s["ids"].copy_(torch.randint(0, 700, (200,), device="cuda"))
        want = [x.clone() for x in _step(K, s)]
        graph, out = graphs[rep % 2]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), rep
        losses.append(want[0].clone())
    assert not torch.equal(losses[0], losses[1])


def test_steps_on_two_streams_at_once():
    """Every call's workspace is its own: two steps in flight on two streams
    give what each gives alone."""
    from pdum_dsl_amd import kernels as K

    cases = [_inputs(300, 256, 900, torch.bfloat16, 1), _inputs(260, 200, 1200, torch.float16, 2)]
    want = [_step(K, s) for s in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = _step(K, cases[i])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
