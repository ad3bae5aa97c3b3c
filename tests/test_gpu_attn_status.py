"""Bounds out of range are reported wherever their sequence stands among many."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_attn_prompt import Case, be  # noqa: F401
from turboqwenfare_amd._lib import ERR_INVALID

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads", [(4, 1, 64), (8, 2, 128), (2, 1, 256), (3, 3, 64)])
@pytest.mark.parametrize("n, at", [(65, 64), (65, 3), (64, 63), (130, 128), (300, 64), (300, 299)])
@pytest.mark.parametrize("queries", [0, 1])
def test_many_short_sequences(be, heads, n, at, queries):  # noqa: F811
    """One row each, so that there are just as many tiles of rows as the totals allow; the bad one has no rows, or one."""
    c = Case(be, [(queries if i == at else 1, 1) for i in range(n)], heads, seed=n)
    good = c.check()
    wrong = np.arange(c.cu_q[at], c.cu_q[min(at + 2, n)])  # its rows, and those of the one that begins where it ends
    rest = np.delete(np.arange(c.tq), wrong)
    for bad in (c.tk + 5, 2 ** 31 - 1, -1):
        cu_k = c.cu_k.copy()
        cu_k[at + 1] = bad
        c.be.write(c.status, np.zeros(1, np.int32))
        got = c.run(d_cu_k=c.dev(cu_k))
        assert c.be.read(c.status, np.int32, (1,))[0] == ERR_INVALID, bad
        assert np.array_equal(got[rest], good[rest])
    c.free()
