"""Prompts of few rows before many keys, whose keys are dealt out and joined: against the definition in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_attn_prompt import Case, be  # noqa: F401
from turboqwenfare_amd._lib import ERR_INVALID

pytestmark = pytest.mark.gpu

HEADS = [(16, 2, 256), (2, 1, 256), (8, 2, 128), (7, 1, 128), (1, 1, 64), (6, 2, 64)]


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("lq, lk", [(1, 3001), (1, 1024), (31, 2048), (33, 2049), (130, 1537), (1100, 1100)])
def test_few_rows_many_keys(be, heads, lq, lk):  # noqa: F811
    c = Case(be, [(lq, lk)], heads, gate=lq % 2 == 1, seed=lq, gaps=(0, 8, 8, 16), behind=(3, 0))
    c.check()
    c.free()


@pytest.mark.parametrize("heads", [(4, 2, 256), (4, 2, 128), (4, 2, 64)])
def test_long_among_short(be, heads):  # noqa: F811
    """Parts without a tile: sequences with no rows, no keys, fewer keys than rows, one key."""
    c = Case(be, [(3, 0), (0, 7), (40, 5001), (1, 1), (0, 0), (40, 9), (70, 4000)], heads, gate=True, seed=21, behind=(5, 3))
    got = c.check()
    assert (got[:3] == 0).all() and (got[44:75] == 0).all()
    c.free()


@pytest.mark.parametrize("heads", [(4, 2, 256), (4, 2, 128), (4, 2, 64)])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
def test_odd_values(be, heads, what):  # noqa: F811
    """In the part that some rows see in part, and in one that all see."""
    def last(c, x):
        x[2][1980, 0, 3] = what
        x[1][1990, 1, 0] = np.nan
    def early(c, x):
        x[2][100, 0, 3] = what
    c = Case(be, [(40, 2000)], heads, seed=22, change=last)
    got = c.check()
    assert np.isfinite(got[:20, :2]).all() and not np.isfinite(got[20:, :2, 3]).any() and np.isnan(got[30:, 2:]).all()
    c.free()
    c = Case(be, [(40, 2000)], heads, seed=22, change=early)
    got = c.check()
    assert not np.isfinite(got[:, :2, 3]).any() and np.isfinite(got[:, 2:]).all()
    c.free()


@pytest.mark.parametrize("heads", [(2, 1, 256), (2, 1, 64)])
def test_sharp_softmax(be, heads):  # noqa: F811
    """Parts whose maxima are far from each other, in each order."""
    for ramp in (np.linspace(0.05, 3.0, 2500), np.linspace(3.0, 0.05, 2500)):
        def change(c, x):
            x[1] *= ramp[:, None, None]
        for sharp in (0.0, 1.0, 40.0):
            c = Case(be, [(37, 2500)], heads, seed=23, sharp=sharp, change=change)
            c.check()
            c.free()


def test_larger_scratch_between(be):  # noqa: F811
    """Calls that cut their keys otherwise, one after another, do not read what the ones before left."""
    a, b = Case(be, [(33, 2049)], (16, 2, 256), seed=24), Case(be, [(200, 6000)], (8, 2, 128), seed=25)
    a.run()
    first = a.raw.copy()
    for _ in range(3):
        b.check()
        a.run()
        assert np.array_equal(a.raw, first)
    a.free(), b.free()


def test_bad_bounds(be):  # noqa: F811
    c = Case(be, [(20, 2000), (30, 3000)], (2, 1, 64), seed=26, behind=(4, 4))
    c.run(d_cu_q=c.dev(np.array([0, 20, 10], np.int32)))
    assert be.read(c.status, np.int32, (1,))[0] == ERR_INVALID
    c.be.write(c.status, np.zeros(1, np.int32))
    c.be.write(c.y, np.full(c.y.nbytes // 2, 0x1234, np.uint16))
    c.check()
    c.free()
