"""Inputs and bounds that the paged-cache tests share."""

import numpy as np

from oracle import paged as op


def batch(rng, lengths, new, page_rows, *, pad=0, spare=2, width=None):
    """A table of pages in any order (-1 behind a sequence's last), starts, lengths, rows and pages of a batch."""
    used = [-(-n // page_rows) for n in lengths]
    width = max([1] + used) + 1 if width is None else width
    pages = sum(used) + spare
    order, at = rng.permutation(pages), 0
    table = np.full((len(lengths), width), -1, dtype=np.int32)
    for i, u in enumerate(used):
        table[i, :u] = order[at : at + u]
        at += u
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    return table, starts, np.array(lengths, dtype=np.int32), int(starts[-1]) + pad, pages


def half(dtype) -> float:
    """The relative error of one rounding to a 16-bit type."""
    return {"bf16": 2.0**-8, "f16": 2.0**-11}[dtype]


def attention_bounds(dtype, o, lse, A, S, V, n, d):
    """How far o and lse may be off, per element.

    x is a sum of d products in fp32 (each of the d additions and the scale
    round by 2^-24 of at most S) and goes through an exp2 of argument x log2 e
    (2^-23 |x| of rounding, 2^-22 of the instruction): a weight is off by the
    factor exp(+-delta), lse by delta and its own sum's roundings. A weight is
    rounded to the type as a factor (half() of it, 2^-25 where f16 runs out of
    exponents: weights are taken over the row's maximum or less, so the sum is
    at least 1), the accumulator rounds 2^-24 an addition and what joins parts
    a few times more, o itself half() of it."""
    delta = (d + 8) * 2.0**-24 * S + 2.0**-22 * S + 2.0**-21
    h = half(dtype)
    tiny = 2.0**-25 if dtype == "f16" else 0.0
    steps = (n + 64) * 2.0**-24
    bo = (h + 2 * delta + 2 * steps + 2.0**-18)[..., None] * A + (tiny * n * V)[..., None]
    bo = bo + h * (np.abs(o) + bo) + (2.0**-25 if dtype == "f16" else 2.0**-133)
    with np.errstate(invalid="ignore"):
        bl = delta + steps + 2.0**-21 + 2.0**-22 * np.abs(np.where(np.isfinite(lse), lse, 0.0))
    return bo, bl


def check_attention(got_o, got_lse, want, dtype, d, what=""):
    o, lse, A, S, V, n = want
    done = ~np.isnan(lse)
    bo, bl = attention_bounds(dtype, o, lse, A, S, V, n, d)
    empty = done & (n == 0)
    assert (got_o[empty] == 0).all() and np.isneginf(got_lse[empty]).all(), f"{what}: rows that see nothing"
    full = done & (n > 0)
    eo, el = np.abs(got_o[full] - o[full]), np.abs(got_lse[full] - lse[full])
    assert np.isfinite(got_o[full]).all(), f"{what}: not finite"
    worst = (eo / bo[full]).max() if eo.size else 0.0
    assert worst <= 1, f"{what}: o is {worst:.2f} of its bound, error {eo.max():.3e}"
    worst = (el / bl[full]).max() if el.size else 0.0
    assert worst <= 1, f"{what}: lse is {worst:.2f} of its bound, error {el.max():.3e}"


__all__ = ["attention_bounds", "batch", "check_attention", "half", "op"]
