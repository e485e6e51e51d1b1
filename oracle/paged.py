"""float64 closed forms of the paged-cache operators: the position rotation,
the 4-bit format, where a token lies, and attention with a window and first
tokens kept. Sequences are walked one by one, rows one by one: nothing here
is shared with the kernels or with the wrappers that call them."""

from __future__ import annotations

import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def rotary_table(positions: int, rotated: int, base: float = 10000.0) -> np.ndarray:
    angle = np.arange(positions)[:, None] * base ** (-np.arange(0, rotated, 2) / rotated)
    return np.concatenate([np.cos(angle), np.sin(angle)], 1).astype(np.float32)


def rotate(x: np.ndarray, row: np.ndarray, interleaved: bool) -> np.ndarray:
    """x [heads, features] turned by one table row, in float32 as it is defined:
    every product and every sum rounded."""
    half = len(row) // 2
    c, s = row[:half].astype(np.float32), row[half:].astype(np.float32)
    x = x.astype(np.float32).copy()
    ia = np.arange(half) * 2 if interleaved else np.arange(half)
    ib = ia + (1 if interleaved else half)
    a, b = x[:, ia], x[:, ib]
    x[:, ia], x[:, ib] = (a * c).astype(np.float32) - (b * s).astype(np.float32), (b * c).astype(np.float32) + (
        a * s).astype(np.float32)
    return x


def fp4(x: np.ndarray, most: int) -> tuple[np.ndarray, np.ndarray]:
    """(codes, scale bytes) of the last axis by groups of 32: every exponent and
    every level is tried in turn."""
    g = np.asarray(x, dtype=np.float64).reshape(-1, 32)
    codes, scales = np.zeros(g.shape, dtype=np.uint8), np.zeros(len(g), dtype=np.uint8)
    for i, row in enumerate(g):
        if not np.isfinite(row).all():
            scales[i] = 255
            continue
        e = next((e for e in range(-126, most) if np.abs(row).max() <= 7.0 * 2.0**e), most)
        scales[i] = e + 127
        for j, v in enumerate(row):
            off = np.abs(LEVELS - abs(v) / 2.0**e)
            near = np.flatnonzero(off == off.min())  # a tie: the even code
            c = int(near[0]) if len(near) == 1 or near[0] % 2 == 0 else int(near[1])
            codes[i, j] = c + (8 if np.signbit(v) else 0)
    lead = x.shape[:-1]
    return codes.reshape(x.shape), scales.reshape(lead + (-1,))


def fp4_values(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """What codes (one an entry) and their groups' bytes stand for."""
    v = np.where(codes & 8, -1.0, 1.0) * LEVELS[codes & 7]
    scale = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return v * np.repeat(scale, 32, axis=-1)


def tokens(starts, lengths, rows: int):
    """(row, sequence, position) of every row that a sequence owns."""
    for i in range(len(lengths)):
        for r in range(max(0, starts[i]), min(rows, starts[i + 1])):
            yield r, i, lengths[i] - (starts[i + 1] - r)


def place(table, i: int, pos: int, page_rows: int, pages: int):
    """(page, row) of a token, None where it has no place."""
    if pos < 0 or pos // page_rows >= table.shape[1]:
        return None
    p = int(table[i, pos // page_rows])
    return (p, pos % page_rows) if 0 <= p < pages else None


def attention(q, k, v, table, starts, lengths, *, scale, window=None, sinks=0, every=1):
    """q [rows, heads_q, features] over pools k, v [pages, heads, page_rows,
    features] of values, all float64. Returns per row and query head o, lse,
    and what the tolerances are made of: A = sum p |v| / den, S = the largest
    scale sum |q k|, n = the number of visible keys, V = their largest |v|. Rows of
    no sequence: o = 0, lse = -inf. Only every ``every``-th row of a sequence,
    and its last, is computed; the others are NaN."""
    rows, hq, d = q.shape
    pages, hkv, pr, _ = k.shape
    o, A = np.zeros((rows, hq, d)), np.zeros((rows, hq, d))
    lse, S, V = np.full((rows, hq), -np.inf), np.zeros((rows, hq)), np.zeros((rows, hq))
    n = np.zeros((rows, hq), dtype=np.int64)
    for r, i, pos in tokens(starts, lengths, rows):
        if (r - starts[i]) % every and r != starts[i + 1] - 1:
            o[r], lse[r] = np.nan, np.nan
            continue
        seen = [s for s in range(pos + 1) if window is None or s > pos - window or s < sinks]
        at = [w for w in (place(table, i, s, pr, pages) for s in seen) if w is not None]
        if not at:
            continue
        pg, off = np.array(at).T
        for h in range(hq):
            kk, vv = k[pg, h // (hq // hkv), off], v[pg, h // (hq // hkv), off]
            with np.errstate(invalid="ignore", over="ignore"):
                x = scale * (kk @ q[r, h])
                m = x.max() if not np.isnan(x).any() else np.nan
                if m == -np.inf:
                    continue
                w = np.exp(x - m)
                den = w.sum()
                o[r, h], lse[r, h] = w @ vv / den, m + np.log(den)
                A[r, h] = w @ np.abs(vv) / den
                S[r, h], V[r, h], n[r, h] = scale * (np.abs(kk) @ np.abs(q[r, h])).max(), np.abs(vv).max(), len(at)
    return o, lse, A, S, V, n
