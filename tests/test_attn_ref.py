"""The attention's definition in 64 bits (attn_ref.py) against loops over its formula, and that its tolerances catch
mistakes (on the CPU)."""
from __future__ import annotations

import math

import numpy as np
import pytest

import attn_ref as ref


def loops(q, k, v, last, scale, gate=None):
    rows, hq, d = q.shape
    y = np.zeros(q.shape)
    for i in range(rows):
        for h in range(hq):
            kh = h // (hq // k.shape[1])
            s = [scale * float(sum(q[i, h, e] * k[j, kh, e] for e in range(d))) for j in range(min(len(k), last[i] + 1))]
            if not s:
                continue
            top = max(s)
            w = [math.exp(a - top) for a in s]
            for j, a in enumerate(w):
                y[i, h] += a / sum(w) * v[j, kh]
            if gate is not None:
                y[i, h] /= 1.0 + np.exp(-gate[i, h])
    return y


def inputs(rows, keys, hq, hk, d, seed=0):
    rng = np.random.default_rng(seed)
    return [rng.standard_normal(s) for s in ((rows, hq, d), (keys, hk, d), (keys, hk, d), (rows, hq, d))]


@pytest.mark.parametrize("rows, keys, hq, hk", [(1, 1, 1, 1), (5, 5, 4, 2), (3, 9, 6, 2), (6, 2, 2, 1), (2, 0, 2, 2)])
def test_against_loops(rows, keys, hq, hk):
    q, k, v, g = inputs(rows, keys, hq, hk, 8)
    last = np.arange(rows) + keys - rows
    for gate in (None, g):
        y, tol = ref.attention(q, k, v, last, 0.3, gate)
        assert np.allclose(y, loops(q, k, v, last, 0.3, gate), rtol=1e-12, atol=1e-14)
        assert (tol >= 0).all()


@pytest.mark.parametrize("keys", [40, 400])
@pytest.mark.parametrize("mistake", ["one key more", "one key less", "scale", "heads", "gate", "no maximum's correction", "values"])
def test_mistakes_are_caught(keys, mistake):
    hq, hk, d, rows = 8, 2, 64, 30
    q, k, v, g = inputs(rows, keys, hq, hk, d, 1)
    last = np.arange(rows) + keys - rows
    want, tol = ref.attention(q, k, v, last, d ** -0.5, g)
    if mistake == "one key more":
        got = loops(q, k, v, np.minimum(last + 1, keys), d ** -0.5, g)
        got[-1] = want[-1]
    elif mistake == "one key less":
        got = loops(q, k, v, last - 1, d ** -0.5, g)
    elif mistake == "scale":
        got = loops(q, k, v, last, 1.1 * d ** -0.5, g)
    elif mistake == "heads":
        got = loops(q[:, np.arange(hq).reshape(-1, hk).T.reshape(-1)], k, v, last, d ** -0.5, g)
    elif mistake == "gate":
        got = loops(q, k, v, last, d ** -0.5)
    elif mistake == "values":
        got = loops(q, k, np.roll(v, 1, 0), last, d ** -0.5, g)
    else:  # what was summed before a larger score is not multiplied down: the first half of the keys weighs double
        got = np.zeros(q.shape)
        for i in range(rows):
            for h in range(hq):
                s = k[:last[i] + 1, h // 4] @ q[i, h] * d ** -0.5
                w = np.exp(s - s.max())
                w[:len(w) // 2] *= 2.0
                got[i, h] = w @ v[:last[i] + 1, h // 4] / w.sum() / (1 + np.exp(-g[i, h]))
    assert (np.abs(got - want) > tol).mean() > 0.02


def test_rounding_to_bf16_is_within_the_tolerance():
    """The definition with its weights and result rounded to bf16, and that tolerance is no more than four such steps."""
    q, k, v, _ = inputs(20, 300, 4, 2, 64, 2)
    last = np.arange(20) + 280
    want, tol = ref.attention(q, k, v, last, 0.125)
    half = lambda x: np.float32(x).astype(np.float64) * (1 + 2.0 ** -8 * np.sign(x) * np.resize([1, -1], x.shape))  # noqa: E731
    got = np.zeros(want.shape)
    for h in range(4):
        s = q[:, h] @ k[:, h // 2].T * 0.125
        s = np.where(np.arange(300) <= last[:, None], s, -np.inf)
        w = np.exp(s - s.max(1, keepdims=True))
        got[:, h] = half(w / w.sum(1, keepdims=True)) @ v[:, h // 2]
    assert (np.abs(half(got) - want) <= tol).all()
    size = np.stack([np.abs(v[:, h // 2]).max() * np.ones((20, 64)) for h in range(4)], 1)
    assert (tol <= 4 * 2.0 ** -8 * size).all()


def test_pages():
    rng = np.random.default_rng(3)
    cache = rng.standard_normal((5, 2, 4, 3))
    rows = ref.gathered(cache, np.array([3, 0, 4]), 10)
    for t in range(10):
        assert np.array_equal(rows[t], cache[[3, 0, 4][t // 4], :, t % 4])


@pytest.mark.parametrize("pairs", ["half", "neighbours"])
def test_rotation_keeps_lengths_and_turns_by_the_distance(pairs):
    """A product of two turned heads depends on the distance of their positions alone."""
    rng = np.random.default_rng(4)
    a, b = rng.standard_normal((2, 1, 1, 16))
    freq = 1e4 ** (-np.arange(6) / 6)
    dots = []
    for first in (0, 5, 100003):
        (x, _), (y, _) = (ref.heads_after(h, None, 0.0, [first + p], freq, pairs) for h, p in ((a, 0), (b, 9)))
        assert np.isclose((x * x).sum(), (a * a).sum())
        dots.append((x * y).sum())
    assert np.allclose(dots, dots[0])


def test_rows_are_divided_by_a_product():
    """The paged kernel's row / group for all of its rows (8 queries of groups of up to 256): row * (2^20 / group + 1) >> 20,
    in 32 bits."""
    for group in range(1, 257):
        row = np.arange(8 * group, dtype=np.uint64)
        product = row * (2 ** 20 // group + 1)
        assert product.max() < 2 ** 32 and np.array_equal(product >> np.uint64(20), row // group)
