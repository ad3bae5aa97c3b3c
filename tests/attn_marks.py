"""Keys and values of which none can be left out or counted twice unseen.

With random values a result shrinks with the root of the keys' number and its tolerance does not, so among thousands of
keys whole tiles may be missing. Here each key's value stands in one dimension alone, that of its stretch of the sequence
(n / d neighbouring keys have one), and is positive: a dimension of y is the weight of its stretch, its tolerance relative
to that, and a few keys more or fewer are a larger part of a stretch than the tolerance is. `ramp` (in units of the
exponent) raises or lowers the scores along the sequence, so that the maximum moves through all of it.
"""
from __future__ import annotations

import numpy as np

import f8_ref

ONE = 8.0  # the queries' first element, which the ramp is multiplied with
RAMPS = {"bf16": (0.0, 20.0, -20.0), "f8": (0.0, 8.0, -8.0)}  # e4m3 has steps of 1/16: a larger one would jump within stretches


def queries(q):
    """q with the ramp's element."""
    q = np.array(q, np.float64)
    q[..., 0] = ONE
    return q


def keys_and_values(rng, n, heads, d, ramp):
    """k, v [n, heads, d] for queries of N(0, 1) and a scale of d^-1/2: scores of N(0, 1/4) and the ramp, -ramp..ramp."""
    k, v = rng.standard_normal((n, heads, d)) * 0.5, np.zeros((n, heads, d))
    if n == 0:
        return k, v
    k[..., 0] = (np.linspace(-ramp, ramp, n) * d ** 0.5 / ONE)[:, None]
    stretch = np.arange(n) * d // max(n, d)
    for h in range(heads):
        v[np.arange(n), h, (stretch + 17 * h) % d] = 1.0 + rng.integers(0, 8, n) / 8.0
    return k, v


def e4m3(x):
    """(bytes, scales f32, values) of rows [..., d], the largest magnitude of each at 448."""
    x = np.asarray(x, np.float64)
    s = (np.abs(x).max(-1) / 448.0).astype(np.float32)
    s[s == 0.0] = 1.0
    z = f8_ref.round_e4m3(x / s[..., None].astype(np.float64))
    b = np.searchsorted(f8_ref.TABLE[:127], np.abs(z)).astype(np.uint8) | np.where(z < 0, 0x80, 0).astype(np.uint8)
    return b, s, f8_ref.TABLE[b] * s[..., None].astype(np.float64)
