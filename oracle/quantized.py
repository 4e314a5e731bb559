"""An 8-bit K/V cache in float64: quantised writes, reads, attention.

Codes are float64 arrays of the values that the 8-bit types can take, so
``codes * scales`` is what a cache stands for, exactly. ``kind`` is "fp8"
(float8 e4m3) or "int8". No counterpart in the reference.
"""

from __future__ import annotations

import numpy as np

MOST = {"fp8": 448.0, "int8": 127.0}


def nearest(x: np.ndarray, kind: str) -> np.ndarray:
    """The nearest code, the even one of two, for |x| up to MOST."""
    x = np.asarray(x, dtype=np.float64)
    if kind == "int8":
        return np.rint(x)
    _, exponent = np.frexp(x)  # |x| in [2^(exponent - 1), 2^exponent)
    step = np.ldexp(1.0, np.maximum(exponent - 1, -6) - 3)
    return np.rint(x / step) * step


def least_scale(most: float, kind: str) -> float:
    """The least power of two s >= 2^-126 with most <= MOST s."""
    s = 2.0 ** -126
    while most > MOST[kind] * s:
        s *= 2
    return s


def append(codes: np.ndarray, scales: np.ndarray, slots, rows: np.ndarray, kind: str) -> None:
    """Write ``rows [T, H, D]`` at ``slots`` into ``codes [N, B, H, D]`` and
    ``scales [N, H]`` in place, one of K and V. Slots outside the pool are
    skipped; of equal ones the last is written."""
    blocks, size, heads, _ = codes.shape
    pages: dict[int, dict[int, int]] = {}
    for t, slot in enumerate(slots):
        if 0 <= slot < blocks * size:
            pages.setdefault(slot // size, {})[slot % size] = t
    for page, at in pages.items():
        first = min(at)
        offsets = sorted(at)
        for h in range(heads):
            x = rows[[at[o] for o in offsets], h].astype(np.float64)
            finite = np.isfinite(x)
            s = least_scale(float(np.abs(x[finite]).max(initial=0.0)), kind)
            if kind == "int8" and not finite.all():
                s = np.nan
            old = scales[page, h]
            if first > 0:
                s = s if np.isnan(s) or old <= s else old
                if s != old and not np.isnan(s):
                    codes[page, :first, h] = nearest(codes[page, :first, h] * (old / s), kind)
            with np.errstate(invalid="ignore"):
                q = nearest(np.where(finite, x / s, 0.0), kind)
            if kind == "fp8":
                q = np.where(finite, q, np.nan)
            codes[page, offsets, h] = np.where(np.isnan(s), 0.0, q) if kind == "int8" else q
            scales[page, h] = s


def gather(codes, scales, tables, contexts) -> np.ndarray:
    """``[sum(contexts), H, D]`` values; rows of invalid blocks are zeros."""
    blocks, size, heads, dim = codes.shape
    out = np.zeros((sum(contexts), heads, dim))
    i = 0
    for table, c in zip(tables, contexts):
        for p in range(c):
            page = table[p // size] if p // size < len(table) else -1
            if 0 <= page < blocks:
                out[i] = codes[page, p % size] * scales[page][:, None]
            i += 1
    return out


def attention(query, k_codes, v_codes, k_scales, v_scales, tables, contexts, cu_q, scale):
    """Causal attention (bottom-right) of the rows of each request over its
    context. Returns the outputs ``[T, Hq, D]`` and what error bounds are made of:
    the same with |v| in place of v, and per row and head the largest scale *
    sum |q k| and the largest weight times its V scale of the positions it sees."""
    query = np.asarray(query, dtype=np.float64)
    blocks, size, hkv, dim = k_codes.shape
    hq = query.shape[1]
    share = hq // hkv
    out, around = np.zeros_like(query), np.zeros_like(query)
    reach, peak = np.zeros((2, *query.shape[:2]))
    for r, c in enumerate(contexts):
        c = min(c, len(tables[r]) * size)
        rows = range(cu_q[r], cu_q[r + 1])
        pos = np.arange(c)
        page = np.asarray(tables[r], dtype=np.int64)[pos // size]
        there = (page >= 0) & (page < blocks)
        pos, page = pos[there], page[there]
        k = k_codes[page, pos % size] * k_scales[page][:, :, None]
        v = v_codes[page, pos % size] * v_scales[page][:, :, None]
        for row in rows:
            seen = pos <= contexts[r] - (cu_q[r + 1] - row)
            if not seen.any():
                continue
            for h in range(hq):
                kk, vv = k[seen, h // share], v[seen, h // share]
                s = scale * (kk @ query[row, h])
                with np.errstate(invalid="ignore"):
                    p = np.exp(s - s.max())
                p /= p.sum()
                out[row, h] = p @ vv
                around[row, h] = p @ np.abs(vv)
                reach[row, h] = abs(scale) * (np.abs(kk) @ np.abs(query[row, h])).max()
                peak[row, h] = (p * v_scales[page[seen], h // share]).max()
    return out, around, reach, peak
