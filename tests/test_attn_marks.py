"""That the long tests of the attentions see a few keys left out or counted twice, wherever they stand (on the CPU: the
mistakes are planted in the definition)."""
from __future__ import annotations

import numpy as np
import pytest

import attn_marks as marks
import attn_ref as ref
import f8_ref


def rounded(x):
    return f8_ref.from_bf16(f8_ref.to_bf16(np.asarray(x, np.float32))).astype(np.float64)


@pytest.mark.parametrize("kind", ["bf16", "f8"])
@pytest.mark.parametrize("ramp", [0, 1, 2], ids=["flat", "up", "down"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n", [300, 3000, 9000, 20000])
def test_blocks_of_keys_are_missed(kind, ramp, d, n):
    rng = np.random.default_rng(n + d)
    k, v = marks.keys_and_values(rng, n, 1, d, marks.RAMPS[kind][ramp])
    k, v = [marks.e4m3(x)[2] for x in (k, v)] if kind == "f8" else [rounded(x) for x in (k, v)]
    q = rounded(marks.queries(rng.standard_normal((1, 1, d))))
    want, tol = (a[0, 0] for a in ref.attention(q, k, v, [n - 1], d ** -0.5))
    s = k[:, 0] @ q[0, 0] * d ** -0.5
    w = np.exp(s - s.max())
    for size in (16, 32, 128):  # a page's slice or an instruction's keys, a wavefront's step, a workgroup's
        at = np.arange(0, n, size)
        block_w, block_v = np.add.reduceat(w, at), np.add.reduceat(w[:, None] * v[:, 0], at, axis=0)
        total_w, total_v = block_w.sum(), block_v.sum(0)
        assert (np.abs(total_v / total_w - want) < 1e-9 * want).all()
        for times in (-1.0, 1.0):
            got = (total_v + times * block_v) / (total_w + times * block_w)[:, None]
            worst = (np.abs(got - want) / tol).max(1)
            assert worst.min() > 1.25, (size, times, int(worst.argmin()), worst.min())


def test_e4m3_rows():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((50, 3, 64)) * np.exp(rng.standard_normal((50, 3, 1)))
    x[4, 1] = 0.0
    b, s, v = marks.e4m3(x)
    assert b.dtype == np.uint8 and s.dtype == np.float32 and not ((b & 127) == 127).any() and (v[4, 1] == 0).all()
    s = s[..., None].astype(np.float64)
    assert (np.abs(v - x) <= s * f8_ref.step(x / s) * 0.51).all()
