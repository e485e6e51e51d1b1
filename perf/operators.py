"""The training operators' measured cases: layer norm with its gradient, dropout from a counter-based generator, and the
softmax cross entropy of a linear head with its gradient, over the range of sizes that training programs call them at.

With ``own`` false ``run`` computes an operator in its plain form, elementary torch operations in 32 bits; with ``own``
true it makes the calls a user makes of ``pdum_dsl_amd.kernels``. ``exact`` is the definition in 64 bits.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5
IGNORE = -100


# ------------------------------------------------------------------ the cases


def _norm(mode, dtype, rows, cols, residual=False, **kw):
    return dict(kind="layernorm", mode=mode, dtype=dtype, rows=rows, cols=cols, residual=residual, **kw)


def _drop(mode, dtype, rows, cols, p, residual=False, **kw):
    return dict(kind="dropout", mode=mode, dtype=dtype, rows=rows, cols=cols, p=p, residual=residual, **kw)


def _loss(mode, dtype, tokens, width, vocab, **kw):
    return dict(kind="loss", mode=mode, dtype=dtype, tokens=tokens, width=width, vocab=vocab, **kw)


def listed() -> list:
    return [
        # a few rows through one norm: latency
        _norm("fwd", "bf16", 64, 768, name="norm_fwd_bf16_64x768"),
        # a block's norm in a 16-bit training step, gpt2-small's width over 8192 tokens, the residual's gradient added
        _norm("train", "bf16", 8192, 768, residual=True, name="norm_train_bf16_8192x768_res"),
        # odd rows and columns: every row starts at another alignment
        _norm("train", "f16", 3001, 1023, name="norm_train_f16_3001x1023"),
        # the row templates' streaming size, with the gradient
        _norm("train", "f32", 8192, 4096, name="norm_train_f32_8192x4096"),
        # an embedding's dropout for a short sequence: latency
        _drop("fwd", "f32", 256, 768, 0.1, name="dropout_fwd_f32_256x768"),
        # a block's residual dropout in a 16-bit training step, forward and backward
        _drop("train", "bf16", 8192, 768, 0.1, residual=True, name="dropout_train_bf16_8192x768_res"),
        # a wide activation of odd width at a high rate
        _drop("train", "f16", 4177, 5003, 0.5, name="dropout_train_f16_4177x5003"),
        # scoring a short text against a small vocabulary: latency
        _loss("fwd", "bf16", 100, 768, 5003, name="loss_fwd_bf16_100x768x5003"),
        # gpt2-small's head and loss in an fp32 training step over one sequence
        _loss("train", "f32", 1024, 768, 50257, name="loss_train_f32_1024x768x50257"),
        # the same head in a 16-bit step over eight sequences
        _loss("train", "bf16", 8192, 768, 50257, name="loss_train_bf16_8192x768x50257"),
        # odd tokens, width and vocabulary
        _loss("train", "f16", 777, 1023, 5003, name="loss_train_f16_777x1023x5003"),
        # a wide model's head: matrix-core throughput
        _loss("train", "bf16", 4096, 4096, 50257, name="loss_train_bf16_4096x4096x50257"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _dtype(rng):
    return rng.choice(("bf16", "bf16", "f16", "f32"))


def _width(rng, lo, hi):
    """Mostly a multiple of 64, as model widths are; a third of them any number."""
    n = _log_int(rng, lo, hi)
    return n if rng.random() < 0.35 else max(64, n // 64 * 64)


def draw(rng) -> dict:
    kind = rng.choice(("layernorm", "dropout", "loss"))
    mode = rng.choice(("fwd", "train", "train"))
    dtype = _dtype(rng)
    while True:
        if kind == "loss":
            tokens, width, vocab = _log_int(rng, 1, 16384), _width(rng, 64, 4096), _log_int(rng, 300, 60000)
            cost = 6.0 * tokens * width * vocab * (6 if dtype == "f32" else 1)
            if cost <= 4.5e12 and tokens * vocab <= 450_000_000:
                return _loss(mode, dtype, tokens, width, vocab)
            continue
        rows, cols = _log_int(rng, 1, 65536), _width(rng, 64, 12000)
        if rows * cols * BYTES[dtype] <= 1 << 27:
            if kind == "layernorm":
                return _norm(mode, dtype, rows, cols, residual=mode == "train" and rng.random() < 0.5)
            return _drop(mode, dtype, rows, cols, rng.choice((0.05, 0.1, 0.2, 0.5)), residual=rng.random() < 0.5)


# ------------------------------------------------------------------ inputs


def _normal(gen, *shape, dtype, std=1.0, mean=0.0):
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    return x.mul_(std).add_(mean).to(dtype)


def _inputs(case, seed) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = TORCH[case["dtype"]]
    if case["kind"] == "loss":
        n, d, v = case["tokens"], case["width"], case["vocab"]
        x = _normal(gen, n, d, dtype=dt)  # the last norm's output
        w = _normal(gen, v, d, dtype=dt, std=2.0 * d**-0.5)  # logits of a standard deviation near 2
        targets = torch.randint(0, v, (n,), generator=gen, device="cuda")
        pad = torch.rand((n,), generator=gen, device="cuda") < 0.05  # padding, which has no loss
        targets = torch.where(pad, torch.full_like(targets, IGNORE), targets)
        live = (targets != IGNORE).to(torch.float32)
        return dict(x=x, w=w, targets=targets, dloss=live / live.sum().clamp(min=1.0))  # the mean's gradient
    r, c = case["rows"], case["cols"]
    if case["kind"] == "layernorm":
        # a residual stream: each feature with an offset and a scale of its own
        off, sc = torch.randn(c, generator=gen, device="cuda"), torch.rand(c, generator=gen, device="cuda") + 0.5
        x = (torch.randn((r, c), generator=gen, device="cuda") * sc + 0.5 * off).to(dt)
        out = dict(x=x, gamma=_normal(gen, c, dtype=dt, std=0.1, mean=1.0), beta=_normal(gen, c, dtype=dt, std=0.1))
        if case["mode"] == "train":
            out["dy"] = _normal(gen, r, c, dtype=dt, std=0.1)
            out["dres"] = _normal(gen, r, c, dtype=dt, std=0.1) if case["residual"] else None
        return out
    out = dict(x=_normal(gen, r, c, dtype=dt), residual=_normal(gen, r, c, dtype=dt) if case["residual"] else None)
    # the generator's seed and the step's number, on the device
    out["rng"] = torch.tensor([seed * 0x9E3779B97F4A7C1 % 2**62, seed % 100000], dtype=torch.int64, device="cuda")
    if case["mode"] == "train":
        out["dy"] = _normal(gen, r, c, dtype=dt, std=0.1)
    return out


def prepare(case, seed):
    return dict(case=case, **_inputs(case, seed))


# ------------------------------------------------------------------ the plain forms


def _plain_layernorm(s):
    x, gamma, dt = s["x"].float(), s["gamma"].float(), s["x"].dtype
    n = x.shape[1]
    mean = x.sum(1) / n
    xc = x - mean[:, None]
    rstd = 1.0 / torch.sqrt((xc * xc).sum(1) / n + EPS)
    xhat = xc * rstd[:, None]
    y = (xhat * gamma + s["beta"].float()).to(dt)
    if s["case"]["mode"] == "fwd":
        return y, mean, rstd
    dy = s["dy"].float()
    u = dy * gamma
    dx = rstd[:, None] * (u - (u.sum(1) / n)[:, None] - xhat * ((u * xhat).sum(1) / n)[:, None])
    if s["dres"] is not None:
        dx = dx + s["dres"].float()
    return y, mean, rstd, dx.to(dt), (dy * xhat).sum(0).to(dt), dy.sum(0).to(dt)


def _plain_keep(rng, rows, cols, threshold, site=0):
    """Philox4x32-10 over 8 consecutive columns a counter, 16 bits each."""
    m32 = 0xFFFFFFFF
    groups = (cols + 7) // 8
    idx = torch.arange(rows * groups, dtype=torch.int64, device=rng.device)
    seed, step = rng[0], rng[1]
    k0, k1 = seed & m32, (seed >> 32) & m32
    c0, c1 = idx & m32, (idx >> 32) & m32
    c2, c3 = (step & m32).expand_as(idx), torch.full_like(idx, site)
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # the 64 bits of the product, as a signed number
        c0, c1, c2, c3 = ((p1 >> 32) & m32) ^ c1 ^ k0, p1 & m32, ((p0 >> 32) & m32) ^ c3 ^ k1, p0 & m32
        k0, k1 = (k0 + 0x9E3779B9) & m32, (k1 + 0xBB67AE85) & m32
    words = torch.stack((c0, c1, c2, c3), 1)
    bits = torch.stack((words & 0xFFFF, words >> 16), 2).reshape(rows, groups * 8)[:, :cols]
    return bits >= threshold


def _plain_dropout(s):
    x, case = s["x"], s["case"]
    threshold = int(round(case["p"] * 65536))
    scale = 65536.0 / (65536 - threshold)
    keep = _plain_keep(s["rng"], x.shape[0], x.shape[1], threshold)
    zero = torch.zeros((), device=x.device)
    y = torch.where(keep, x.float() * scale, zero)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    if case["mode"] == "fwd":
        return y.to(x.dtype)
    keep = _plain_keep(s["rng"], x.shape[0], x.shape[1], threshold)  # the mask is never stored
    return y.to(x.dtype), torch.where(keep, s["dy"].float() * scale, zero).to(x.dtype)


def _plain_loss(s):
    x, w, targets = s["x"].float(), s["w"].float(), s["targets"]
    live = targets != IGNORE
    col = torch.where(live, targets, torch.zeros_like(targets))[:, None]
    z = x @ w.t()
    mx = z.max(1, keepdim=True).values
    lse = torch.log(torch.exp(z - mx).sum(1)) + mx[:, 0]
    loss = torch.where(live, lse - z.gather(1, col)[:, 0], torch.zeros_like(lse))
    if s["case"]["mode"] == "fwd":
        return loss, lse
    g = torch.where(live, s["dloss"], torch.zeros_like(lse))[:, None]
    dz = torch.exp(z - lse[:, None])
    dz.scatter_add_(1, col, torch.full_like(col, -1, dtype=torch.float32))
    dz = dz * g
    return loss, lse, (dz @ w).to(s["x"].dtype), (dz.t() @ x).to(s["w"].dtype)


# ------------------------------------------------------------------ one pass


def _own(s):
    from pdum_dsl_amd import kernels as K

    case = s["case"]
    train = case["mode"] == "train"
    if case["kind"] == "layernorm":
        f = K.layernorm_fwd(s["x"], s["gamma"], s["beta"], EPS)
        if not train:
            return f.y, f.mean, f.rstd
        return (f.y, f.mean, f.rstd) + K.layernorm_bwd(s["x"], s["dy"], f.mean, f.rstd, s["gamma"], dres=s["dres"])
    if case["kind"] == "dropout":
        y = K.dropout_fwd(s["x"], case["p"], s["rng"], residual=s["residual"])
        return (y, K.dropout_bwd(s["dy"], case["p"], s["rng"])) if train else y
    f = K.linear_cross_entropy(s["x"], s["w"], s["targets"], ignore_index=IGNORE)
    if not train:
        return f.loss, f.lse
    return (f.loss, f.lse) + K.linear_cross_entropy_bwd(s["x"], s["w"], s["targets"], f.lse, s["dloss"],
                                                        ignore_index=IGNORE)


def run(state):
    if own:
        return _own(state)
    return {"layernorm": _plain_layernorm, "dropout": _plain_dropout, "loss": _plain_loss}[state["case"]["kind"]](state)


# ------------------------------------------------------------------ what a pass cannot do without


def work(case) -> dict:
    es = BYTES[case["dtype"]]
    train = case["mode"] == "train"
    if case["kind"] == "loss":
        n, d, v = case["tokens"], case["width"], case["vocab"]
        once = (n * d + v * d) * es + 8 * n + 8 * n  # x, w, targets; loss and lse
        return dict(bytes=once + ((n * d + v * d) * es + 4 * n if train else 0),
                    flops=(6 if train else 2) * n * v * d)
    r, c, more = case["rows"], case["cols"], 1 if case["residual"] else 0
    if case["kind"] == "layernorm":
        b = 2 * r * c * es + 2 * c * es + 8 * r  # x, y; gamma and beta; the statistics
        if train:
            b += (2 + more) * r * c * es + 2 * c * es  # dy and dx (x is read already); the weights' gradients
        return dict(bytes=b, flops=(8 + (14 if train else 0)) * r * c)
    passes = 2 + more + (2 if train else 0)
    # ten rounds of four multiplications and six other operations for eight elements, each way
    return dict(bytes=passes * r * c * es, flops=(2 if train else 1) * 14 * r * c)


# ------------------------------------------------------------------ the definitions in 64 bits


def _exact_layernorm(s):
    x, g, b = (s[k].double() for k in ("x", "gamma", "beta"))
    mean = x.mean(dim=-1, keepdim=True)
    var = ((x - mean) ** 2).mean(dim=-1, keepdim=True)
    rstd = (var + EPS) ** -0.5
    norm = (x - mean) * rstd
    out = [norm * g + b, mean[:, 0], rstd[:, 0]]
    if s["case"]["mode"] == "train":
        dy = s["dy"].double()
        dn = dy * g
        dx = (dn - dn.mean(-1, keepdim=True) - norm * (dn * norm).mean(-1, keepdim=True)) * rstd
        out += [dx if s["dres"] is None else dx + s["dres"].double(), (dy * norm).sum(0), dy.sum(0)]
    return tuple(out)


def _exact_mask(seed, step, rows, cols, p):
    """The same generator in numpy's unsigned words."""
    per_row = -(-cols // 8)
    n = np.arange(rows * per_row, dtype=np.uint64)
    mask = np.uint64(2**32 - 1)
    s32 = np.uint64(32)
    ctr = [n & mask, n >> s32, np.full_like(n, step % 2**32), np.zeros_like(n)]
    key = [seed % 2**32, seed >> 32]
    for _ in range(10):
        a, b = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
        ctr = [(b >> s32) ^ ctr[1] ^ np.uint64(key[0]), b & mask, (a >> s32) ^ ctr[3] ^ np.uint64(key[1]), a & mask]
        key = [(key[0] + 0x9E3779B9) % 2**32, (key[1] + 0xBB67AE85) % 2**32]
    words = np.stack(ctr, axis=1).astype("<u4")
    bits = words.view("<u2").reshape(rows, per_row * 8)
    return bits[:, :cols] >= round(p * 65536)


def _exact_dropout(s):
    case = s["case"]
    seed, step = (int(v) for v in s["rng"].tolist())
    keep = torch.from_numpy(_exact_mask(seed, step, case["rows"], case["cols"], case["p"])).to(s["x"].device)
    scale = 65536 / (65536 - round(case["p"] * 65536))
    y = torch.zeros(keep.shape, dtype=torch.float64, device=keep.device)
    y[keep] = s["x"].double()[keep] * scale
    if s["residual"] is not None:
        y += s["residual"].double()
    if case["mode"] == "fwd":
        return y
    dx = torch.zeros_like(y)
    dx[keep] = s["dy"].double()[keep] * scale
    return y, dx


def _exact_loss(s):
    w, targets = s["w"].double(), s["targets"]
    n, d = s["x"].shape
    train = s["case"]["mode"] == "train"
    loss = torch.zeros(n, dtype=torch.float64, device=w.device)
    lse = torch.zeros_like(loss)
    dx = torch.zeros((n, d), dtype=torch.float64, device=w.device)
    dw = torch.zeros_like(w) if train else None
    for lo in range(0, n, 1024):  # the logits of 1024 tokens at a time
        at = slice(lo, min(n, lo + 1024))
        x, t = s["x"][at].double(), targets[at]
        z = torch.mm(x, w.T)
        lse[at] = torch.logsumexp(z, dim=1)
        rows = torch.nonzero(t != IGNORE)[:, 0]
        loss[at][rows] = lse[at][rows] - z[rows, t[rows]]
        if train:
            p = torch.softmax(z, dim=1)
            p[rows, t[rows]] -= 1.0
            g = torch.zeros(x.shape[0], dtype=torch.float64, device=w.device)
            g[rows] = s["dloss"][at][rows].double()
            p *= g[:, None]
            dx[at] = torch.mm(p, w)
            dw += torch.mm(p.T, x)
    return (loss, lse, dx, dw) if train else (loss, lse)


def exact(case, seed):
    s = prepare(case, seed)
    return {"layernorm": _exact_layernorm, "dropout": _exact_dropout, "loss": _exact_loss}[case["kind"]](s)
