"""Plain statements in 64 bits of the heads' norms and rotation and of the two
attentions, and the tolerances that their arithmetic gives."""
from __future__ import annotations

import numpy as np

import f8_ref

BF16, F32 = 2.0 ** -8, 2.0 ** -24  # half a step, relative


# ---- norms and rotation --------------------------------------------------------------
def heads_after(x, w, eps, positions, freq, pairs):
    """x [t, heads, d] f64 -> (value, tolerance of its f32 arithmetic) after the norm (w None: none) and the rotation."""
    d = x.shape[2]
    if w is not None:
        with np.errstate(divide="ignore", invalid="ignore"):  # a zero row with eps 0
            x = x / np.sqrt((x * x).mean(2, keepdims=True) + eps) * w.astype(np.float64)
    # the norm's f32 sum of d squares and a handful of roundings; the angle is 64-bit up to half a turn, then f32:
    # 2^-25 turns and the two functions' last bits
    tol = np.abs(x) * ((d + 16) * F32 if w is not None else 0.0)
    n = len(freq)
    if n == 0:
        return x, tol
    a = np.asarray(positions, np.float64)[:, None] * np.asarray(freq, np.float64)
    c, s = np.cos(a)[:, None], np.sin(a)[:, None]
    i, j = (slice(0, n), slice(n, 2 * n)) if pairs == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    out, otol = x.copy(), tol.copy()
    out[..., i], out[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
    both = np.abs(x[..., i]) + np.abs(x[..., j])
    otol[..., i] = otol[..., j] = both * ((d + 16) * F32 + 2.0 ** -21)
    return out, otol


# ---- attention -------------------------------------------------------------------------
def attention(q, k, v, last, scale, gate=None):
    """q [rows, q_heads, d], k and v [keys, kv_heads, d] f64, last [rows]: the last key that a row sees (below 0: none)
    -> (y, tolerance of a bf16 y whose weights are bf16 and whose sums are f32)."""
    rows, hq, d = q.shape
    keys, hk = k.shape[0], k.shape[1]
    y, tol = np.zeros(q.shape), np.zeros(q.shape)
    seen = np.arange(keys)[None, :] <= np.asarray(last)[:, None]
    for h in range(hq):
        kk, vv = k[:, h // (hq // hk)], v[:, h // (hq // hk)]
        # rows with the same keys together, so that what others see stays out of their products
        groups = [np.arange(rows)] if np.isfinite(kk).all() and np.isfinite(vv).all() else [np.array([r]) for r in range(rows)]
        for r in groups:
            at = seen[r].any(0)
            if not at.any():
                continue
            with np.errstate(all="ignore"):
                dot = q[r, h] @ kk[at].T
                s = np.where(seen[r][:, at], dot * scale, -np.inf)
                top = s.max(1, keepdims=True)
                p = np.exp(s - np.where(top == -np.inf, 0.0, top))
                total = p.sum(1, keepdims=True)
                p = p / np.where(total == 0.0, 1.0, total)
                y[r, h], size = p @ vv[at], p @ np.abs(vv[at])
                # a score's f32 dot product, and its two roundings before and in the exponential
                ds = np.where(seen[r][:, at], (np.abs(q[r, h]) @ np.abs(kk[at]).T * scale * (d + 4) + np.abs(dot) * scale * 4) * F32, 0.0).max(1, keepdims=True)
            n = int(at.sum())
            # the weights' rounding; exponentials (2^-22); sums of n terms; a rescaling at most once in 32 keys, twice the
            # error of a score (numerator and sum)
            tol[r, h] = size * (BF16 + 2.0 ** -21 + (n + n / 16 + 16) * F32 + 2 * ds)
    if gate is not None:
        f = 1.0 / (1.0 + np.exp(-gate))
        y, tol = y * f, tol * f + np.abs(y * f) * 2.0 ** -20
    return y, tol + (np.abs(y) + tol) * BF16 + 2.0 ** -126


def prompt(q, k, v, cu_q, cu_k, scale, gate=None):
    """The same for packed sequences; rows outside them are NaN in both."""
    y, tol = np.full(q.shape, np.nan), np.full(q.shape, np.nan)
    for a, b, c, e in zip(cu_q[:-1], cu_q[1:], cu_k[:-1], cu_k[1:]):
        last = np.arange(b - a) + (e - c) - (b - a)
        y[a:b], tol[a:b] = attention(q[a:b], k[c:e], v[c:e], last, scale, None if gate is None else gate[a:b])
    return y, tol


def gathered(cache, table, n):
    """Tokens 0..n of a sequence out of a cache [pages, heads, page, d] -> [n, heads, d]."""
    page = cache.shape[2]
    ids = table[:-(-n // page)]
    return cache[ids].transpose(0, 2, 1, 3).reshape(-1, cache.shape[1], cache.shape[3])[:n]


def paged(q, k, v, table, lens, rows, scale, gate=None):
    y, tol = np.zeros(q.shape), np.zeros(q.shape)
    for s, n in enumerate(lens):
        at = slice(s * rows, (s + 1) * rows)
        y[at], tol[at] = attention(q[at], gathered(k, table[s], n), gathered(v, table[s], n), np.arange(rows) + n - rows, scale,
                                   None if gate is None else gate[at])
    return y, tol


# ---- the e4m3 cache ----------------------------------------------------------------------
def f8_cache(rng, shape):
    """(bytes, scales, values f64) of a random e4m3 cache [pages, heads, page, d]."""
    b = rng.integers(0, 256, shape).astype(np.uint8)
    b[(b & 127) == 127] ^= 1
    s = (rng.uniform(0.5, 1.5, shape[:3]) / 150.0).astype(np.float32)
    return b, s, f8_ref.TABLE[b] * s[..., None].astype(np.float64)
