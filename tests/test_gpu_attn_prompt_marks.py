"""Prompt attention over thousands of keys of which none can be left out or counted twice unseen (attn_marks.py), whole and
dealt out to several workgroups, against the definition in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

import attn_marks as marks
from test_gpu_attn_prompt import Case, be  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ramp", [0, 1, 2], ids=["flat", "up", "down"])
@pytest.mark.parametrize("heads", [(4, 2, 256), (4, 1, 128), (3, 1, 64)])
@pytest.mark.parametrize("seqs", [[(1, 9000)], [(40, 5001)], [(512, 4096)], [(1100, 1100)], [(300, 1500), (700, 700), (1, 2049), (33, 3000)],
                                  [(9, 9)] * 40 + [(70, 3000)]], ids=lambda s: "+".join("%dx%d" % x for x in s[-2:]))
def test_keys_are_counted_once(be, heads, seqs, ramp):  # noqa: F811
    def change(c, x):
        rng = np.random.default_rng(1)
        x[0] = marks.queries(x[0])
        for a, b in zip(c.cu_k[:-1], c.cu_k[1:]):
            x[1][a:b], x[2][a:b] = marks.keys_and_values(rng, b - a, heads[1], heads[2], marks.RAMPS["bf16"][ramp])

    c = Case(be, seqs, heads, gate=len(seqs) > 1, seed=30, change=change)
    c.check()
    c.free()
