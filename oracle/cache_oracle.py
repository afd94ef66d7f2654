"""64-bit restatement of the latent-cache operators (cache_write, cache_read, tree_attn,
verify_draft) in numpy, written from their definitions: the checks' side of
tests/test_cache_gpu.py, tests/test_tree_attn_gpu.py and tests/test_verify_gpu.py.

The reference implements none of the four; the row scale is the "ue8m0" format its
ModelArgs name (baseline/indexer.py:15).
"""
from __future__ import annotations

import numpy as np


def e4m3_values() -> np.ndarray:
    """The value of each of the 256 e4m3 codes (sign, 4 exponent bits with bias 7, 3 mantissa
    bits; no infinities, NaN at 0x7F and 0xFF)."""
    code = np.arange(256)
    e, m = (code >> 3) & 15, code & 7
    v = np.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * 2.0 ** (e - 7.0))
    v = np.where(code >= 128, -v, v)
    v[[0x7F, 0xFF]] = np.nan
    return v


def e4m3_codes(x: np.ndarray) -> np.ndarray:
    """Nearest e4m3 code of finite x (saturating at 448), ties to the even mantissa."""
    grid = e4m3_values()[:0x7F]  # non-negative codes ascend in value
    a = np.abs(x)
    hi = np.clip(np.searchsorted(grid, a), 0, 0x7E)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - grid[lo], grid[hi] - a
    take_lo = (dl < dh) | ((dl == dh) & (lo % 2 == 0))
    return (np.where(take_lo, lo, hi) | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def row_scale(x: np.ndarray) -> np.ndarray:
    """Smallest power of two >= max(max |x|, 1e-4) / 448 of each row, at most 2^119."""
    v = np.maximum(np.abs(x).max(-1), np.float64(np.float32(1e-4))) / 448.0
    m, e = np.frexp(v)
    return np.ldexp(1.0, np.minimum(np.where(m == 0.5, e - 1, e), 119))


def cache_rows(x: np.ndarray, dq: int):
    """(codes, scale) of rows x [R, D] (float64 values of bf16 rows); rows with a NaN or an
    infinity get zero codes and scale NaN."""
    bad = ~np.isfinite(x).all(-1)
    safe = np.where(bad[:, None], 0.0, x[:, :dq])
    s = row_scale(safe)
    codes = e4m3_codes(safe / s[:, None])
    codes[bad] = 0
    return codes, np.where(bad, np.nan, s)


def sequence_rows(codes, scale, tail, table, n):
    """float64 rows [n, D] of one sequence: codes [slots, dq], scale [slots], tail
    [slots, dr] or None, table [pages] of that sequence and the page size in table[1]."""
    pages, page = table
    pos = np.arange(n)
    slot = np.asarray(pages, np.int64)[pos // page] * page + pos % page
    x = e4m3_values()[codes[slot]] * scale[slot].astype(np.float64)[:, None]
    if tail is not None:
        x = np.concatenate([x, tail[slot].astype(np.float64)], 1)
    x[np.isnan(scale[slot])] = np.nan  # a marked row, its tail too
    return x


def tree_attn_row(q, rows, seen, scale, sink, dv):
    """One drafted token of one sequence: q [H, D], rows [N, D], seen bool [N].  Returns
    (out [H, dv], the same sums over |v|: the scale of the rounding errors)."""
    rows = rows[seen]
    s = q @ rows.T * scale                                    # [H, n]
    top = s.max(1, initial=-np.inf) if sink is None else np.maximum(s.max(1, initial=-np.inf), sink)
    top = np.where(np.isneginf(top), 0.0, top)
    e = np.exp(s - top[:, None])
    den = e.sum(1) + (0.0 if sink is None else np.exp(sink - top))
    den = np.where(den == 0, 1.0, den)
    w = e / den[:, None]
    return w @ rows[:, :dv], w @ np.abs(rows[:, :dv])


def next_token(w, p, noise):
    """argmax of w / noise in single precision, ties to the lowest; p where w is all zero."""
    if not (w > 0).any():
        w = p
    return int(np.argmax(w.astype(np.float32) / noise.astype(np.float32)))


def verify_chain(p, q, tokens, u, noise):
    """One sequence, sampled chain: (out tokens, path)."""
    f = np.float32
    for i, x in enumerate(tokens):
        ok = 0 <= x < p.shape[1] and f(u[i]) * f(q[i, x]) < f(p[i, x])
        if not ok:
            w = np.maximum(p[i] - q[i], f(0))
            return list(tokens[:i]) + [next_token(w, p[i], noise)], list(range(i))
    return list(tokens) + [next_token(p[len(tokens)], p[len(tokens)], noise)], list(range(len(tokens)))


def verify_tree(p, tokens, parents, u, noise):
    """One sequence, fixed candidates: (out tokens, path)."""
    V, row, out, path = p.shape[1], 0, [], []
    while True:
        kids = [i for i in range(len(tokens)) if parents[i] == row - 1 and parents[i] < i and 0 <= tokens[i] < V]
        at, used, taken = 0.0, set(), None
        for i in kids:
            if tokens[i] in used:
                continue
            used.add(tokens[i])
            step = float(p[row, tokens[i]])
            if at <= float(u[row]) < at + step:
                taken = i
            at += step
        if taken is None:
            w = p[row].copy()
            w[[tokens[i] for i in kids]] = 0
            return out + [next_token(w, p[row], noise)], path
        out.append(tokens[taken])
        path.append(taken)
        row = taken + 1
