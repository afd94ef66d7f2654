"""64-bit restatement of the operators over the per-head cache (kv_append, kv_attn) and of
token_logprobs in numpy, written from their definitions: the checks' side of
tests/test_kv_append_gpu.py, tests/test_kv_attn_gpu.py and tests/test_logprobs_gpu.py.

The reference implements none of them; the scales are the "ue8m0" format its ModelArgs
name (baseline/indexer.py:15).
"""
from __future__ import annotations

import numpy as np

from .cache_oracle import e4m3_codes, e4m3_values


def scale_of(amax: np.ndarray) -> np.ndarray:
    """Smallest power of two >= max(amax, 1e-4) / 448, at most 2^119."""
    v = np.maximum(amax, np.float64(np.float32(1e-4))) / 448.0
    m, e = np.frexp(v)
    return np.ldexp(1.0, np.minimum(np.where(m == 0.5, e - 1, e), 119))


def rotate(x: np.ndarray, freqs, rows: np.ndarray) -> np.ndarray:
    """x [n, heads, D] (values of bf16), the last 2 * freqs.shape[1] columns as pairs rotated
    by freqs[rows]; each product and sum rounded to fp32, as the operator defines it."""
    x = np.array(x, np.float32)
    if freqs is None or freqs.shape[1] == 0:
        return x
    rd = 2 * freqs.shape[1]
    f = np.asarray(freqs, np.float32)[np.clip(rows, 0, freqs.shape[0] - 1)][:, None]
    a, b = x[..., -rd::2].copy(), x[..., x.shape[-1] - rd + 1::2].copy()
    x[..., -rd::2] = a * f[..., 0] - b * f[..., 1]
    x[..., x.shape[-1] - rd + 1::2] = a * f[..., 1] + b * f[..., 0]
    return x


def append(x, codes, scale, table, length, block):
    """Rows x [n, heads, D] (fp32 values) of one sequence appended in place to codes uint8
    [pages, heads, page, D] and scale float64 [pages, heads, page / block]."""
    page, n = codes.shape[2], x.shape[0]
    at = length
    while at < length + n:
        stop = min(length + n, (at // block + 1) * block)
        p, r = int(table[at // page]), at % page
        rows = np.moveaxis(x[at - length: stop - length].astype(np.float64), 0, 1)  # [heads, rows, D]
        bad = ~np.isfinite(rows)
        s = scale_of(np.abs(np.where(bad, 0.0, rows)).max((1, 2)))
        mark = bad.any((1, 2))
        first, k = r // block * block, r // block
        if at % block:
            old, was = unmarked(scale[p, :, k])
            s = np.maximum(s, old)
            mark |= was
            kept = codes[p, :, first:r]
            v = e4m3_values()[kept] * (old / s)[:, None, None]
            nan = np.isnan(v)
            codes[p, :, first:r] = np.where(nan, kept, e4m3_codes(np.where(nan, 0.0, v)))
        c = e4m3_codes(np.where(bad, 0.0, rows) / s[:, None, None])
        codes[p, :, r:r + stop - at] = np.where(bad, 0x7F, c)
        scale[p, :, k] = np.where(mark, s * (1 + 2.0 ** -23), s)
        at = stop


def unmarked(scale):
    """(power of two, marked) of scales as kv_append leaves them."""
    m, e = np.frexp(np.asarray(scale, np.float64))
    return np.where(m == 0, 0.0, np.ldexp(1.0, e - 1)), (m != 0.5) & (m != 0)


def head_rows(codes, scale, table, n):
    """float64 [n, heads, D]: the first n positions of a sequence."""
    page = codes.shape[2]
    block = page // scale.shape[2]
    pos = np.arange(n)
    p, r = np.asarray(table, np.int64)[pos // page], pos % page
    return e4m3_values()[codes[p, :, r]] * unmarked(scale[p, :, r // block])[0][..., None]


def attn_token(q, k, v, seen, scale, sink):
    """One token of one sequence: q [H, D], k, v [n, heads, D], seen bool [n].  Returns
    (out [H, D], the same sums over |v|: the scale of the rounding errors)."""
    H, heads = q.shape[0], k.shape[1]
    k, v = k[seen], v[seen]
    out, size = np.zeros((H, v.shape[2])), np.zeros((H, v.shape[2]))
    with np.errstate(invalid="ignore", over="ignore"):
        for h in range(H):
            g = h // (H // heads)
            s = k[:, g] @ q[h] * scale
            top = max(s.max(initial=-np.inf), -np.inf if sink is None else sink[h])
            if np.isnan(s).any():
                out[h] = size[h] = np.nan
                continue
            top = 0.0 if np.isneginf(top) else top
            e = np.exp(s - top)
            den = e.sum() + (0.0 if sink is None else np.exp(sink[h] - top))
            w = e / (den if den else 1.0)
            out[h], size[h] = w @ v[:, g], w @ np.abs(v[:, g])
    return out, size


def logprobs(x, token, top):
    """One row of logits in float64: (logp, entropy, top_logp, top_ids)."""
    m = x.max()
    if not np.isfinite(m) or np.isnan(x).any():
        lse = ent = np.nan
    else:
        e = np.exp(x - m)
        lse = m + np.log(e.sum())
        with np.errstate(invalid="ignore"):
            ent = np.where(e > 0, e * (m - x), 0.0).sum() / e.sum() + np.log(e.sum())
    # NaN above all, then by value, the lowest index first
    key = np.where(np.isnan(x), np.inf, x)
    ids = np.lexsort((np.arange(x.size), -key, ~np.isnan(x)))[:top]
    return (0.0 if token < 0 else x[token] - lse), ent, x[ids] - lse, ids
