"""TEST INFRASTRUCTURE ONLY -- float64 numpy restatement of the 8-bit paged KV cache.

Only tests/ may import this module. Codes are e4m3 values (held here as float64), scales powers of
two, one for each block of 16 tokens and head; arrays are [pages, kv_heads, page, head_dim] and
[pages, kv_heads, page / 16] (one layer).
"""
from __future__ import annotations

import numpy as np

BLOCK = 16


def e4m3(x):
    """The e4m3 value nearest to x (ties to the even code), saturating at 448; from the format:
    3 mantissa bits, exponents -6 .. 8, subnormals down to 2^-9."""
    x = np.asarray(x, np.float64)
    a = np.abs(x)
    _, e = np.frexp(np.where(a > 0, a, 1.0))
    step = np.exp2(np.maximum(e - 1, -6) - 3)
    with np.errstate(invalid="ignore"):
        r = np.minimum(np.rint(a / step) * step, 448.0)
    return np.where(np.isnan(x), np.nan, np.copysign(r, x))


def scale_of(amax: float) -> float:
    """The smallest power of two, at least 2^-120, of which amax is at most 448 times."""
    s = 2.0 ** -120
    if amax > 448.0 * s:
        s = 2.0 ** np.ceil(np.log2(amax / 448.0))
        while amax > 448.0 * s:
            s *= 2
        while amax <= 448.0 * (s / 2):
            s /= 2
    return s


def rope(x, cs):
    """x [heads, dim] by the angles cs [dim / 2, 2]."""
    x0, x1, c, s = x[..., 0::2], x[..., 1::2], cs[:, 0], cs[:, 1]
    out = np.empty_like(x)
    out[..., 0::2], out[..., 1::2] = x0 * c - x1 * s, x0 * s + x1 * c
    return out


def append(codes, scales, new, table_row, start):
    """Writes new [n, kv_heads, dim] at positions start .. into (codes, scales), in place. Infinite
    values do not count for the scale (and saturate)."""
    page = codes.shape[2]
    n, done = new.shape[0], 0
    while done < n:
        pos = start + done
        take = min(n - done, BLOCK - pos % BLOCK)
        pg = table_row[pos // page] if pos // page < len(table_row) else -1
        blk, slot = pos % page // BLOCK, pos % BLOCK
        if 0 <= pg < codes.shape[0]:
            for h in range(codes.shape[1]):
                x = new[done:done + take, h]
                s = scale_of(float(np.max(np.where(np.isfinite(x), np.abs(x), 0.0))))
                rows = codes[pg, h, blk * BLOCK:(blk + 1) * BLOCK]
                if slot:
                    old = scales[pg, h, blk]
                    s = max(s, old)
                    rows[:slot] = e4m3(rows[:slot] * (old / s))
                rows[slot:slot + take] = e4m3(x / s)
                scales[pg, h, blk] = s
        done += take


def values(codes, scales):
    return codes * np.repeat(scales, BLOCK, axis=2)[..., None]


def attention(q, k_vals, v_vals, table_row, length, first_pos, window=0, sinks=0, scale=None):
    """q [n, heads, dim] at positions first_pos ..; k_vals, v_vals [pages, kv_heads, page, dim]."""
    n, heads, dim = q.shape
    pages, kv, page, _ = k_vals.shape
    scale = dim ** -0.5 if scale is None else scale
    out = np.zeros((n, heads, dim))
    for i in range(n):
        p = first_pos + i
        seen = [j for j in range(min(length, p + 1)) if (window == 0 or j > p - window or j < sinks)
                and j // page < len(table_row) and 0 <= table_row[j // page] < pages]
        if not seen:
            continue
        pg = np.array([table_row[j // page] for j in seen])
        at = np.array(seen) % page
        for h in range(heads):
            k, v = k_vals[pg, h // (heads // kv), at], v_vals[pg, h // (heads // kv), at]
            s = k @ q[i, h] * scale
            w = np.exp(s - s.max())
            out[i, h] = (w / w.sum()) @ v
    return out
