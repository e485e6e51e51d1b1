"""The serving operators' measured cases: appending to a paged cache of keys and values with the position rotation on the
way, and attention over that cache, held in 16 or in 4 bits, with and without a sliding window beside first tokens that
stay visible; from one token a sequence to whole prompts.

With ``own`` false ``run`` computes an operator in its plain form, elementary torch operations in 32 bits; with ``own``
true it makes the calls a user makes of ``pdum_dsl_amd.kernels``. ``exact`` is the definition in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

TORCH = {"bf16": torch.bfloat16, "f16": torch.float16}
GROUP = 32  # features that share a 4-bit cache's scale
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # the magnitudes of the 4-bit codes


# ------------------------------------------------------------------ the cases


def _append(dtype, bits, batch, tokens, keys, heads_q, heads_kv, dim, page, **kw):
    """``batch`` sequences of up to ``keys`` tokens, the last up to ``tokens`` of each new."""
    case = dict(kind="append", dtype=dtype, bits=bits, batch=batch, tokens=tokens, keys=keys, heads_q=heads_q,
                heads_kv=heads_kv, dim=dim, page=page, rotated=dim, interleaved=False, ragged=False, pad=0)
    return {**case, **kw}


def _attend(dtype, bits, batch, tokens, keys, heads_q, heads_kv, dim, page, **kw):
    """``tokens`` query tokens a sequence over up to ``keys`` keys; window 0: none."""
    case = dict(kind="attend", dtype=dtype, bits=bits, batch=batch, tokens=tokens, keys=keys, heads_q=heads_q,
                heads_kv=heads_kv, dim=dim, page=page, window=0, sinks=0, ragged=False, pad=0)
    return {**case, **kw}


def listed() -> list:
    return [
        # one step of 64 sequences: a token each, latency
        _append("bf16", 16, 64, 1, 1000, 32, 8, 128, 16, ragged=True, name="append_bf16_64x1"),
        # eight prompts go into the cache
        _append("bf16", 16, 8, 1024, 1024, 32, 8, 128, 16, name="append_bf16_8x1024"),
        # the same prompts into a cache of 4 bits, read back as attention sees it
        _append("bf16", 4, 8, 1024, 1024, 32, 8, 128, 32, name="append4_bf16_8x1024"),
        # odd pieces of prompts, half of the features rotated, in neighbouring pairs, and rows of no sequence
        _append("f16", 4, 5, 77, 1001, 12, 12, 64, 64, rotated=32, interleaved=True, ragged=True, pad=19,
                name="append4_f16_5x77_pairs"),
        # one user's next token: latency
        _attend("bf16", 16, 1, 1, 1000, 32, 8, 128, 16, name="decode_bf16_1x1000"),
        # the grouped-query decode workload over a paged cache: bandwidth
        _attend("bf16", 16, 64, 1, 8192, 32, 8, 128, 16, name="decode_bf16_64x8192"),
        # long sequences of different lengths of which a window and the first tokens are read
        _attend("f16", 16, 24, 1, 30000, 32, 8, 128, 64, window=4096, sinks=4, ragged=True, name="decode_f16_24x30000_window"),
        # the decode workload over a cache of 4 bits
        _attend("bf16", 4, 64, 1, 8192, 32, 8, 128, 16, name="decode4_bf16_64x8192"),
        # a few drafted tokens of some sequences, over 4 bits
        _attend("f16", 4, 7, 4, 5003, 12, 12, 64, 32, ragged=True, pad=3, name="draft4_f16_7x4x5003"),
        # a prompt of the attention workload's length
        _attend("bf16", 16, 2, 4096, 4096, 32, 8, 128, 16, name="prompt_bf16_2x4096"),
        # a long prompt under a window with first tokens kept
        _attend("bf16", 16, 1, 8192, 8192, 32, 8, 128, 64, window=1024, sinks=4, name="prompt_bf16_8192_window"),
        # the next piece of some prompts over a cache of 4 bits, odd lengths
        _attend("bf16", 4, 4, 500, 7001, 32, 8, 128, 16, ragged=True, name="piece4_bf16_4x500x7001"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    while True:
        kind = rng.choice(("append", "attend", "attend"))
        dtype, bits = rng.choice(("bf16", "bf16", "f16")), rng.choice((16, 16, 4))
        heads_q, heads_kv, dim = rng.choice(((32, 8, 128), (32, 8, 128), (12, 12, 64), (16, 4, 64), (16, 1, 128), (8, 8, 128)))
        page = rng.choice((16, 32, 64, 128))
        batch = _log_int(rng, 1, 96)
        keys = _log_int(rng, 1, 32768)
        tokens = 1 if rng.random() < 0.5 else _log_int(rng, 1, 8192)
        tokens = min(tokens, keys)
        ragged, pad = rng.random() < 0.6, rng.choice((0, 0, 0, 1, 37))
        if batch * keys * heads_kv * dim > 64 * 8192 * 8 * 128 or batch * tokens > 16384:
            continue
        sizes = (dtype, bits, batch, tokens, keys, heads_q, heads_kv, dim, page)
        if kind == "append":
            rotated = rng.choice((dim, dim, dim // 2))
            return _append(*sizes, rotated=rotated, interleaved=rng.random() < 0.3, ragged=ragged, pad=pad)
        if batch * tokens * keys * heads_q > 2 * 4096 * 4096 * 32:
            continue
        window, sinks = rng.choice(((0, 0), (0, 0), (_log_int(rng, 16, 8192), rng.choice((0, 1, 4, 50)))))
        return _attend(*sizes, window=window, sinks=sinks, ragged=ragged, pad=pad)


def _spread(case):
    """Each sequence's (new tokens, tokens in the cache): all alike, or ragged down to one token and half of the keys."""
    b, t, k = case["batch"], case["tokens"], case["keys"]
    if not case["ragged"]:
        return [t] * b, [k] * b
    lengths = [max(1, k - (i * 37 % b) * k // (2 * b)) for i in range(b)]
    new = [min(max(1, t - (i * 13 % b) * t // b), n) for i, n in enumerate(lengths)]
    return new, lengths


# ------------------------------------------------------------------ inputs


def _normal(gen, *shape, dtype, std=1.0):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).mul_(std).to(dtype)


def _outliers(gen, heads, dim):
    """Keys hold a few features that are larger than the others throughout."""
    wide = torch.rand((heads, 1, dim), generator=gen, device="cuda") < 0.04
    return torch.where(wide, 4.0, 1.0)


def _rotary(positions, rotated):
    """cos, then sin, of every position's angles."""
    inv = 10000.0 ** (-torch.arange(0, rotated, 2, dtype=torch.float64, device="cuda") / rotated)
    angles = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.cat((torch.cos(angles), torch.sin(angles)), 1).float()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, b, page, dim = TORCH[case["dtype"]], case["batch"], case["page"], case["dim"]
    hq, hkv = case["heads_q"], case["heads_kv"]
    new, lengths = _spread(case)
    used = [-(-n // page) for n in lengths]
    width = max(used) + 1
    pages = sum(used) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)  # pages lie anywhere in the pool
    firsts = torch.tensor([sum(used[:i]) for i in range(b)], device="cuda")[:, None] + torch.arange(width, device="cuda")
    live = torch.arange(width, device="cuda") < torch.tensor(used, device="cuda")[:, None]
    table = torch.where(live, order[firsts.clamp(max=pages - 1)], torch.full_like(firsts, -1).to(torch.int32))
    starts = torch.tensor([sum(new[:i]) for i in range(b + 1)], dtype=torch.int32, device="cuda")
    rows = sum(new) + case["pad"]
    wide = _outliers(gen, hkv, dim)
    k, v = _normal(gen, pages, hkv, page, dim, dtype=dt), _normal(gen, pages, hkv, page, dim, dtype=dt)
    k.mul_(wide.to(dt))
    s = dict(case=case, table=table, starts=starts, lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"),
             rows=rows, most=max(new), k=k, v=v, k_scale=None, v_scale=None)
    if case["bits"] == 4:
        s["k"], s["k_scale"] = _quantised(k, case["dtype"])
        s["v"], s["v_scale"] = _quantised(v, case["dtype"])
    s["q"] = _normal(gen, rows, hq, dim, dtype=dt)
    if case["kind"] == "append":
        s["new_k"] = _normal(gen, rows, hkv, dim, dtype=dt).mul_(wide[:, 0].to(dt))
        s["new_v"] = _normal(gen, rows, hkv, dim, dtype=dt)
        s["rotary"] = _rotary(max(lengths), case["rotated"])
    return s


# ------------------------------------------------------------------ the plain forms


def _quantised(x, dtype):
    """x in 4 bits, two codes a byte, and each group's scale 2^(byte - 127), the least that leaves no value over 7."""
    g = x.float().unflatten(-1, (-1, GROUP))
    m, ex = torch.frexp(g.abs().amax(-1))
    e = torch.where(m <= 0.875, ex - 3, ex - 2).clamp(-126, 13 if dtype == "f16" else 127)
    a = torch.ldexp(g.abs(), -e[..., None])
    code = sum(((a > 0.25).byte(), (a >= 0.75).byte(), (a > 1.25).byte(), (a >= 1.75).byte(), (a > 2.5).byte(),
                (a >= 3.5).byte(), (a > 5.0).byte()))  # the nearest level, of two the one with the even code
    code = (code + 8 * (g < 0).byte()).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).byte()


def _values(codes, scale):
    """What a 4-bit tensor stands for, in 32 bits."""
    if scale is None:
        return codes.float()
    levels = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=codes.device)
    x = torch.stack((levels[(codes & 15).int()], levels[(codes >> 4).int()]), -1).flatten(-2)
    return torch.ldexp(x.unflatten(-1, (-1, GROUP)), (scale.int() - 127)[..., None]).flatten(-2)


def _places(s):
    """Each row's sequence and position; rows of no sequence are left out."""
    row = torch.arange(s["rows"], device=s["starts"].device)
    seq = torch.searchsorted(s["starts"][1:].long(), row, right=True)
    row, seq = row[seq < s["case"]["batch"]], seq[seq < s["case"]["batch"]]
    return row, seq, s["lengths"][seq] - s["starts"][seq + 1] + row


def _plain_rotate(x, rotary, pos, case):
    rot = case["rotated"]
    c, sn = rotary[pos][:, None, : rot // 2], rotary[pos][:, None, rot // 2 :]
    x = x.float()
    if case["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack((a * c - b * sn, b * c + a * sn), -1).flatten(-2)
    else:
        a, b = x[..., : rot // 2], x[..., rot // 2 : rot]
        y = torch.cat((a * c - b * sn, b * c + a * sn), -1)
    return torch.cat((y, x[..., rot:]), -1)


def _plain_append(s):
    case, dt = s["case"], s["q"].dtype
    row, seq, pos = _places(s)
    page, off = s["table"][seq, pos // case["page"]].long(), pos % case["page"]
    k = _plain_rotate(s["new_k"][row], s["rotary"], pos, case)
    v = s["new_v"][row].float()
    q = torch.zeros_like(s["q"])
    q[row] = _plain_rotate(s["q"][row], s["rotary"], pos, case).to(dt)
    if case["bits"] == 16:
        s["k"][page, :, off] = k.to(dt)
        s["v"][page, :, off] = v.to(dt)
        return s["k"], s["v"], q
    s["k"][page, :, off], s["k_scale"][page, :, off] = _quantised(k, case["dtype"])
    s["v"][page, :, off], s["v_scale"][page, :, off] = _quantised(v, case["dtype"])
    out = torch.zeros((2,) + s["new_k"].shape, dtype=dt, device=q.device)
    out[0, row] = _values(s["k"][page, :, off], s["k_scale"][page, :, off]).to(dt)
    out[1, row] = _values(s["v"][page, :, off], s["v_scale"][page, :, off]).to(dt)
    return out[0], out[1], q


def _plain_attend(s):
    case = s["case"]
    b, t, hq, hkv, dim = case["batch"], s["most"], case["heads_q"], case["heads_kv"], case["dim"]
    at = s["table"].clamp(min=0).long()

    def cached(codes, scale):  # [batch, heads, keys, features]
        x = _values(codes[at], None if scale is None else scale[at])
        return x.transpose(1, 2).flatten(2, 3)

    k, v = cached(s["k"], s["k_scale"]), cached(s["v"], s["v_scale"])
    keys = k.shape[2]
    new = s["starts"][1:] - s["starts"][:-1]
    j = torch.arange(t, device=new.device)
    row = (s["starts"][:-1, None] + j).clamp(max=s["rows"] - 1)
    q = s["q"][row].float().transpose(1, 2).reshape(b, hkv, hq // hkv * t, dim)
    x = (torch.matmul(q, k.transpose(-1, -2)) * dim**-0.5).view(b, hq, t, keys)
    pos = (s["lengths"] - new)[:, None] + j
    key = torch.arange(keys, device=new.device)
    seen = key <= pos[..., None]
    if case["window"]:
        seen &= (key > pos[..., None] - case["window"]) | (key < case["sinks"])
    x.masked_fill_(~seen[:, None], -math.inf)
    mx = x.amax(-1, keepdim=True)
    p = x.sub_(mx).exp_()
    den = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(b, hkv, -1, keys), v).view(b, hq, t, dim) / den
    lse = (mx + torch.log(den))[..., 0]
    live = j < new[:, None]
    out = torch.zeros_like(s["q"])
    out_lse = torch.full((s["rows"], hq), -math.inf, device=out.device)
    out[row[live]] = o.transpose(1, 2)[live].to(out.dtype)
    out_lse[row[live]] = lse.transpose(1, 2)[live]
    return out, out_lse


# ------------------------------------------------------------------ one pass


def _own(s):
    from pdum_dsl_amd import kernels as K

    case = s["case"]
    if "cache" not in s:  # a program keeps its cache from step to step
        s["cache"] = K.PagedCache(s["k"], s["v"], s["k_scale"], s["v_scale"], TORCH[case["dtype"]])
    cache = s["cache"]
    if case["kind"] == "attend":
        return K.paged_attention(s["q"], cache, s["table"], s["starts"], s["lengths"], window=case["window"] or None,
                                 sinks=case["sinks"])
    q = K.paged_append(s["new_k"], s["new_v"], cache, s["table"], s["starts"], s["lengths"], q=s["q"], rotary=s["rotary"],
                       interleaved=case["interleaved"])
    if case["bits"] == 16:
        return s["k"], s["v"], q
    return K.paged_rows(cache, s["table"], s["starts"], s["lengths"], s["rows"]) + (q,)


def run(state):
    if own:
        return _own(state)
    return _plain_append(state) if state["case"]["kind"] == "append" else _plain_attend(state)


# ------------------------------------------------------------------ what a pass cannot do without


def work(case) -> dict:
    new, lengths = _spread(case)
    rows, hq, hkv, dim = sum(new), case["heads_q"], case["heads_kv"], case["dim"]
    held = 2.0 if case["bits"] == 16 else 0.5 + 1.0 / GROUP  # bytes of a cached element
    if case["kind"] == "append":
        back = 0 if case["bits"] == 16 else rows * 2 * hkv * dim * (held + 2)  # read back as values
        return dict(bytes=rows * dim * (2 * hq * 2 + 2 * hkv * (2 + held)) + 4 * rows * case["rotated"] + back,
                    flops=3 * rows * (hq + hkv) * case["rotated"])
    window, sinks = case["window"] or 1 << 60, case["sinks"]
    read = pairs = 0
    for t, n in zip(new, lengths):
        first = max(0, n - t - window + 1)  # of the window of the first row
        read += n - first + min(sinks, first)
        for p in range(n - t, n):
            lo = max(0, p - window + 1)
            pairs += p - lo + 1 + min(sinks, lo)
    return dict(bytes=int(read * 2 * hkv * dim * held + rows * hq * (dim * 4 + 4)), flops=4 * dim * hq * pairs)


# ------------------------------------------------------------------ the definitions in 64 bits


def _exact_codes(x, dtype):
    """The values that 4 bits hold of x."""
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    top = g.abs().max(dim=-1, keepdim=True).values
    e = torch.ceil(torch.log2(top.clamp(min=1e-300) / 7)).clamp(-126, 13 if dtype == "f16" else 127)
    e = torch.where(7 * torch.exp2(e - 1) >= top, e - 1, torch.where(7 * torch.exp2(e) < top, e + 1, e))
    e = e.clamp(-126, 13 if dtype == "f16" else 127)
    a = g.abs() / torch.exp2(e)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    a = (torch.round(a / step) * step).clamp(max=6.0)
    return (torch.sign(g) * a * torch.exp2(e)).reshape(x.shape)


def _exact_append(s):
    case = s["case"]
    rot, page = case["rotated"], case["page"]
    new, lengths = _spread(case)
    keys, values, q = s["new_k"].double(), s["new_v"].double(), s["q"].double()
    table = s["table"].tolist()
    first = torch.arange(0, rot, 2) if case["interleaved"] else torch.arange(rot // 2)
    second = first + (1 if case["interleaved"] else rot // 2)
    pos = [n - t + j for t, n in zip(new, lengths) for j in range(t)]
    angle = s["rotary"].double()[torch.tensor(pos, device=q.device)]
    turn = torch.complex(angle[:, : rot // 2], angle[:, rot // 2 :])[:, None]
    rows = len(pos)
    for x in (keys, q):
        y = torch.complex(x[:rows][..., first], x[:rows][..., second]) * turn
        x[:rows, :, first], x[:rows, :, second] = y.real, y.imag
        if x is q:
            x[rows:] = 0
    if case["bits"] == 4:
        keys, values = _exact_codes(keys, case["dtype"]), _exact_codes(values, case["dtype"])
        keys[rows:] = 0
        values[rows:] = 0
        return keys, values, q
    k, v = s["k"].double(), s["v"].double()
    place = torch.tensor([table[i][p // page] * page + p % page
                          for i, (t, n) in enumerate(zip(new, lengths)) for p in range(n - t, n)], device=q.device)
    k[place // page, :, place % page] = keys[:rows]
    v[place // page, :, place % page] = values[:rows]
    return k, v, q


def _exact_attend(s):
    case = s["case"]
    hq, hkv, dim = case["heads_q"], case["heads_kv"], case["dim"]
    new, lengths = _spread(case)
    if sum(t * n for t, n in zip(new, lengths)) * hq * dim > 3e11:
        return None
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device=o.device)
    half = torch.tensor([0, 1, 2, 3, 4, 6, 8, 12], dtype=torch.float64, device=o.device) / 2

    def held(name, pages, h, n):  # the first n keys' (values') rows of one head
        x = s[name][pages, h]
        if case["bits"] == 16:
            return x.double().reshape(-1, dim)[:n]
        both = torch.stack((x % 16, x // 16), dim=-1).reshape(-1, dim)[:n].long()
        unit = torch.exp2(s[name + "_scale"][pages, h].double() - 127).reshape(-1, dim // GROUP)[:n]
        return torch.where(both < 8, 1.0, -1.0) * half[both % 8] * unit.repeat_interleave(GROUP, dim=1)

    at = 0
    for i, (t, n) in enumerate(zip(new, lengths)):
        pages = s["table"][i, : -(-n // case["page"])].long()
        p = torch.arange(n - t, n, device=o.device)[:, None]
        key = torch.arange(n, device=o.device)[None]
        hidden = key > p
        if case["window"]:
            hidden = hidden | ((p - key >= case["window"]) & (key >= case["sinks"]))
        for h in range(hkv):
            k, v = held("k", pages, h, n), held("v", pages, h, n)
            for head in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                z = (s["q"][at : at + t, head].double() @ k.T) / math.sqrt(dim)
                z[hidden] = -math.inf
                o[at : at + t, head] = torch.softmax(z, dim=1) @ v
                lse[at : at + t, head] = torch.logsumexp(z, dim=1)
        at += t
    return o, lse


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_append(s) if case["kind"] == "append" else _exact_attend(s)
