"""Rows that see no key are 0 whatever stands in their gates, as padding has anything there."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_attn_paged import Case as Paged
from test_gpu_attn_prompt import Case as Prompt, be, bf16  # noqa: F401

pytestmark = pytest.mark.gpu

HEADS = [(16, 2, 256), (8, 2, 128), (6, 2, 64), (1, 1, 64)]


def odd_gates(shape, rows, seed):
    """Gates [t, heads, d + gap] of which those of `rows` are NaN, infinities or anything."""
    g = np.random.default_rng(seed).standard_normal(shape)
    for i, r in enumerate(rows):
        g[r] = [np.nan, np.inf, -np.inf, 3e38][i % 4]
        g[r, :, ::7] = np.nan
    return g


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("seqs", [[(5, 5), (33, 0), (40, 7), (129, 129), (1, 300), (3, 2)], [(40, 9), (70, 4000), (3, 0), (40, 5001)]], ids=["whole", "parts"])
def test_prompts(be, heads, seqs):  # noqa: F811
    none, at = [], 0
    for lq, lk in seqs:
        none += range(at, at + max(0, lq - lk))
        at += lq

    def change(c, x):
        x[3] = odd_gates(x[3].shape, none, 1)

    c = Prompt(be, seqs, heads, gate=True, seed=2, gaps=(0, 0, 0, 8), change=change)
    c.gate[none] = 0.0  # their factor does not matter
    got = c.check()
    assert none and (got[none] == 0).all()
    c.free()


@pytest.mark.parametrize("kind", ["bf16", "f8"])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("rows", [3, 8])
def test_rows_over_the_cache(be, kind, heads, rows):  # noqa: F811
    """Alone, so that the workgroup writes them, and in a batch."""
    for lens in ([2], [0, 1, 700, 2, 0, 2500, 5] * 3):
        none = [s * rows + i for s, n in enumerate(lens) for i in range(max(0, rows - n))]
        c = Paged(be, lens, rows, heads, kind, gate=True, seed=3, gap=8)
        nq, _, d = heads
        bits, g = bf16(odd_gates((len(lens) * rows, nq, d + 8), none, 4))
        c.gate = g[..., :d].copy()
        c.gate[none] = 0.0
        c.args["d_gate"] = c.dev(bits)
        got = c.check()
        assert (got[none] == 0).all()
        c.free()
