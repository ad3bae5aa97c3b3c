"""Plain statements in 64 bits of the e4m3 block-128 products and of the
router, and the tolerances that their arithmetic gives."""
from __future__ import annotations

import numpy as np

NONE = 0xFFFF
TINY = 2.0 ** -100


# ---- the format ---------------------------------------------------------------------
def e4m3_table() -> np.ndarray:
    """The 256 values: sign, four exponent bits (bias 7), three of fraction; 0x7F and 0xFF are NaN."""
    b = np.arange(256)
    ex, fr = (b >> 3) & 15, b & 7
    v = np.where(ex == 0, fr / 8.0 * 2.0 ** -6, (1 + fr / 8.0) * 2.0 ** (ex - 7.0))
    v = np.where((b & 127) == 127, np.nan, v)
    return np.where(b >= 128, -v, v)


TABLE = e4m3_table()


def step(z) -> np.ndarray:
    """The distance between e4m3 neighbours around |z|."""
    a = np.maximum(np.abs(z), 2.0 ** -6)
    return 2.0 ** (np.minimum(np.floor(np.log2(a)), 8) - 3)


def round_e4m3(z) -> np.ndarray:
    """To nearest, ties to even, for |z| <= 448 and a rounding."""
    z = np.asarray(z, np.float64)
    u = step(z)
    return np.clip(np.rint(z / u) * u, -448, 448)


def quantize(x):
    """Rows [t, n] f32 -> (q [t, n], scale [t, n], z [t, n]): the values, the scale each has, and what was rounded."""
    x = np.asarray(x, np.float32)
    t, n = x.shape
    p = np.zeros((t, -(-n // 128) * 128), np.float32)
    p[:, :n] = x
    p = p.reshape(t, -1, 128)
    a = np.abs(p).max(2, keepdims=True)
    zero = a < np.float32(TINY)
    with np.errstate(divide="ignore", over="ignore", invalid="ignore"):
        s = np.where(zero, np.float32(0), a / np.float32(448))
        inv = np.where(zero, np.float32(0), np.float32(448) / a)
        z = (p * inv).astype(np.float32).astype(np.float64)
    q = round_e4m3(z)
    full = lambda v: np.broadcast_to(v, p.shape).reshape(t, -1)[:, :n].astype(np.float64)  # noqa: E731
    return full(q), full(s), full(z)


def random_matrix(rng, rows, cols, spread=0):
    """(bytes [rows, cols], scales [blocks, blocks]) of a matrix of size cols^-1/2; spread: scales over 2^-spread..1."""
    b = rng.integers(0, 256, (rows, cols)).astype(np.uint8)
    b[(b & 127) == 127] ^= 1
    s = rng.uniform(0.5, 1.0, (-(-rows // 128), -(-cols // 128))) * cols ** -0.5 / 120.0
    s *= 2.0 ** -rng.integers(0, spread + 1, s.shape)
    return b, s.astype(np.float32)


def values(b, s) -> np.ndarray:
    rows, cols = b.shape
    return TABLE[b] * np.repeat(np.repeat(s.astype(np.float64), 128, 0)[:rows], 128, 1)[:, :cols]


def to_bf16(x) -> np.ndarray:
    """f32 -> bf16 bits, to nearest, ties to even."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def from_bf16(b) -> np.ndarray:
    return (np.ascontiguousarray(b, np.uint16).astype(np.uint32) << 16).view(np.float32)


# ---- products -------------------------------------------------------------------------
# Products of a block on the bf16 cores are exact, their sums f32 (an add loses at most a step of the partial sum, so
# 128 of them 128 * 2^-23 of the block's magnitudes).  The fp8 cores take eight products at a time and cut each to a
# grid of 2^-13 of the largest one's power of two (test_how_the_fp8_cores_cut_products): a product loses less than
# 2^-13 of the largest, which itself loses nothing, so the eight less than 7 * 2^-13 of their sum of magnitudes, and so
# does the block.  (Random blocks lose 1.3e-5 of it, seldom more than 2^-14.)  Then per block a rounding of the scale
# and of the fma.
EXACT_BLOCK = 128 * 2.0 ** -23
FP8_BLOCK = 7 * 2.0 ** -13


def block_error(cols, fp8):
    return (FP8_BLOCK if fp8 else 0) + EXACT_BLOCK + (4 * -(-cols // 128) + 4) * 2.0 ** -23


def rounding(kind):
    return 2.0 ** -8 if kind == "bf16" else 2.0 ** -24


def matmul(x, w, fp8):
    """Rows x (f32 values) times the matrix w [rows, cols] in 64 bits: (y, how far f32 arithmetic may be from it)."""
    q, s, _ = quantize(x)
    v = q * s
    return v @ w.T, block_error(w.shape[1], fp8) * (np.abs(v) @ np.abs(w).T)


def experts(x, ids, weights, mats, fp8, kind):
    """(y, tolerance) of the routed experts; mats: for each expert (gate, up, down) in 64 bits.

    h is quantised again, so where its rounding decides, an error before it may move a value by a whole step: the
    values of h within their own error of the middle of two steps are counted as moved."""
    y, tol = np.zeros((x.shape[0], mats[0][2].shape[0])), np.zeros((x.shape[0], mats[0][2].shape[0]))
    for e in np.unique(ids):
        if e == NONE:
            continue
        rows, slot = np.nonzero(ids == e)
        gate, up, down = mats[e]
        (g, dg), (u, du) = matmul(x[rows], gate, fp8), matmul(x[rows], up, fp8)
        sg = g / (1 + np.exp(-g))
        h = sg * u
        # |silu'| <= 1.1; exp, the reciprocal and the products: a few roundings of 2^-22 each
        dh = 1.1 * dg * np.abs(u) + np.abs(sg) * du + 1.1 * dg * du + 2.0 ** -19 * np.abs(h)
        q, s, z = quantize(h)
        top = s * 448
        rel = np.zeros_like(h)  # the error of the block's largest value, as a share of it
        for at in range(0, h.shape[1], 128):
            b = slice(at, at + 128)
            big = np.maximum(top[:, at:at + 1], 1e-300)
            rel[:, b] = (dh[:, b].max(1, keepdims=True) / big) + 2.0 ** -22
        with np.errstate(divide="ignore", invalid="ignore"):
            dz = np.where(s > 0, dh / np.maximum(s, 1e-300), 0) + np.abs(z) * rel
        lo, hi = round_e4m3(z - dz), round_e4m3(z + dz)
        moved = np.maximum(hi - q, q - lo) * s + np.abs(q) * s * rel
        v = q * s
        part, dpart = v @ down.T, moved @ np.abs(down).T + block_error(down.shape[1], fp8) * ((np.abs(v) + moved) @ np.abs(down).T)
        wt = weights[rows, slot].astype(np.float64)[:, None]
        np.add.at(y, rows, wt * part)
        np.add.at(tol, rows, np.abs(wt) * (dpart + ids.shape[1] * 2.0 ** -23 * np.abs(part)))
    return y, tol + rounding(kind) * (np.abs(y) + tol)


# ---- routes ------------------------------------------------------------------------------
def route(logits, top_k, score="softmax", bias=None, n_groups=1, top_groups=1, group_best=1, renormalise=True, scale=1.0):
    """(ids, w, failed rows) from the definition, one row at a time."""
    lg = np.asarray(logits, np.float64)
    t, n = lg.shape
    ids, w, failed = np.full((t, top_k), NONE, np.uint16), np.zeros((t, top_k)), []
    size = n // n_groups
    for r in range(t):
        l = lg[r]
        live = l != -np.inf
        if np.isnan(l).any() or (l == np.inf).any():
            failed.append(r)
            continue
        s = np.zeros(n)
        if live.any():
            if score == "softmax":
                s[live] = np.exp(l[live] - l[live].max())
                s /= s.sum()
            else:
                with np.errstate(over="ignore"):
                    s[live] = 1 / (1 + np.exp(-l[live]))
        c = np.where(live, s + (0 if bias is None else np.asarray(bias, np.float64)), -np.inf)
        if np.isnan(c).any() or (c == np.inf).any():
            failed.append(r)
            continue
        if n_groups > 1:
            total = []
            for g in range(n_groups):
                best = sorted((v for v in c[g * size:(g + 1) * size] if v > -np.inf), reverse=True)[:group_best]
                total.append(sum(best) if best else -np.inf)
            for g in sorted(range(n_groups), key=lambda g: (-total[g], g))[top_groups:]:
                c[g * size:(g + 1) * size] = -np.inf
        pick = [e for e in sorted(range(n), key=lambda e: (-c[e], e))[:top_k] if c[e] > -np.inf]
        p = s[pick]
        if renormalise:
            p = p / p.sum() if p.sum() > 0 else 0 * p
        ids[r, :len(pick)], w[r, :len(pick)] = pick, p * float(np.float32(scale))
    return ids, w, failed
