"""F8 products of up to 16 rows: exact within a block for both types of y, also where the quantised rows do not fit a
workgroup's LDS."""
from __future__ import annotations

import numpy as np
import pytest

import f8_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    from turboqwenfare_amd.backend import HipBackend

    with HipBackend(0) as b:
        yield b


def cancelling(rng, t, rows, cols):
    """(x [t, cols] f32, e4m3 bytes [rows, cols], y [t, rows]).  In every block two products of 448 x 448 cancel and, in
    up to eight blocks, the first and the last among them, six small ones stand beside them: integers below 2^24, so
    that y is exact in f32 in any order, and lost where products are cut to 2^-13 of their neighbours."""
    code = {v: int(np.flatnonzero(ref.TABLE == v)[0]) for v in (448.0, -448.0, 1.0, 2.0)}
    blocks = cols // 128
    x, q = np.zeros((t, cols), np.float32), np.zeros((rows, cols), np.uint8)
    x[:, 0::128] = x[:, 1::128] = 448
    q[:, 0::128], q[:, 1::128] = code[448.0], code[-448.0]
    y = np.zeros((t, rows))
    for b in np.unique(np.r_[0, blocks - 1, rng.integers(0, blocks, 6)]):
        small = rng.integers(0, 3, (rows, 6))
        x[:, b * 128 + 2:b * 128 + 8] = few = rng.integers(1, 4, (t, 6))
        q[:, b * 128 + 2:b * 128 + 8] = np.choose(small, [0, code[1.0], code[2.0]])
        y += few @ small.T
    return x, q, y


# 16 rows of 6912 columns, 15 of 7296 and 2 of 55552 are the most that a workgroup's LDS takes
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("t,rows,cols", [
    (16, 40, 6912), (16, 130, 7040), (16, 40, 7168), (15, 40, 7296), (15, 257, 7424), (14, 40, 8192), (15, 40, 8192), (16, 1000, 8192),
    (2, 40, 55552), (2, 40, 55680), (2, 40, 65536), (1, 40, 65536), (16, 130, 65536), (16, 33000, 7040)])
def test_up_to_16_rows_are_exact(be, t, rows, cols, kind):
    x, q, want = cancelling(np.random.default_rng(t + rows + cols), t, rows, cols)
    w = be.upload_f8(q, np.ones((-(-rows // 128), cols // 128), np.float32))
    d_x = be.to_device(ref.to_bf16(x) if kind == "bf16" else x)
    for y_kind in ("f32", "bf16"):
        d_y = be.to_device(np.full((t, rows), 7, np.uint16 if y_kind == "bf16" else np.float32))
        be.f8_matmul_device(w, d_x, t, d_y, x_type=kind, y_type=y_kind)
        if y_kind == "f32":
            assert np.array_equal(be.read(d_y, np.float32, (t, rows)), want)
        else:
            assert np.array_equal(be.read(d_y, np.uint16, (t, rows)), ref.to_bf16(want.astype(np.float32)))
        be.free(d_y)
    be.free(d_x)
    be.free_weights(w)
