"""F8 products of small integers, whose results are exact whatever cores and sums make them: a product that is left out,
taken twice or scaled by another block's number shows in every form, over many blocks of K."""
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


def integers(rng, t, rows, cols):
    """(x f32, e4m3 bytes, scales, y f32) with x of -7..7 (or twice that), a 7 in each block of each row, so that its
    scale is 2^-6 or 2^-5, and weights of -4..4 under scales of 1, 2 and 4.  All sums are of integers and stay below 2^24,
    and no product is 2^13 times one of its neighbours, so that the fp8 cores keep all."""
    codes = np.array([int(np.flatnonzero(ref.TABLE == v)[0]) for v in range(-4, 5)], np.uint8)
    br, bc = -(-rows // 128), -(-cols // 128)
    x = rng.integers(-7, 8, (t, cols)).astype(np.float32)
    for b in range(bc):
        n = min(128, cols - b * 128)
        x[np.arange(t), b * 128 + rng.integers(0, n, t)] = np.where(rng.random(t) < 0.5, 7, -7)
        x[:, b * 128:b * 128 + n] *= 2.0 ** rng.integers(0, 2, (t, 1))
    at = rng.integers(0, 9, (rows, cols), dtype=np.uint8)
    s = 2.0 ** rng.integers(0, 3, (br, bc))
    w = (at.astype(np.float32) - 4) * np.repeat(np.repeat(s, 128, 0)[:rows], 128, 1)[:, :cols].astype(np.float32)
    assert cols * 14 * 16 < 1 << 24
    return x, codes[at], s.astype(np.float32), x @ w.T


def check(be, t, rows, cols, y_kinds=("f32", "bf16")):
    x, q, s, want = integers(np.random.default_rng(t + 3 * rows + 7 * cols), t, rows, cols)
    w = be.upload_f8(q, s)
    for kind, y_kind in zip(("bf16", "f32"), y_kinds):
        d_x = be.to_device(ref.to_bf16(x) if kind == "bf16" else x)
        bt = np.uint16 if y_kind == "bf16" else np.float32
        d_y = be.to_device(np.full((t, rows), 7, bt))
        be.f8_matmul_device(w, d_x, t, d_y, x_type=kind, y_type=y_kind)
        got = be.read(d_y, bt, (t, rows))
        right = ref.to_bf16(want) if y_kind == "bf16" else want
        assert np.array_equal(got, right), (y_kind, np.argwhere(got != right)[:4], (got != right).sum())
        be.free(d_x)
        be.free(d_y)
    be.free_weights(w)


# few rows; K split over wavefronts, 32, 64 and 128 rows to a workgroup; with fewer K blocks than wavefronts and more
@pytest.mark.parametrize("t,rows,cols", [
    (1, 512, 2048), (3, 100, 1500), (16, 40000, 300), (16, 257, 4000), (17, 300, 2048), (32, 1000, 1300), (50, 512, 2100), (64, 4000, 1920),
    (100, 700, 4095), (300, 1024, 2177), (512, 4096, 1100)])
def test_few_rows_and_split_k(be, t, rows, cols):
    check(be, t, rows, cols)


# Tiles.  A matrix of 8200 rows: 900 rows are tiles of 64, 1900 of 96, 1500 of 256 (and f32 results of 64); of 33000:
# 32 and 64 rows.  Numbers of K blocks of each remainder by the two and three stages of the tiles' loops.
@pytest.mark.parametrize("cols", [100, 256, 1920, 2048, 2100, 2300])
@pytest.mark.parametrize("t,rows", [(900, 8200), (1900, 8200), (1500, 8200), (2300, 8000)])
def test_tiles_over_many_blocks(be, t, rows, cols):
    check(be, t, rows, cols)


@pytest.mark.parametrize("cols", [129, 700, 1024, 1153])
@pytest.mark.parametrize("t", [20, 60, 129, 257])
def test_tiles_of_a_tall_matrix(be, t, cols):
    check(be, t, 33001, cols)


@pytest.mark.parametrize("t,rows,cols", [(900, 8200, 2100), (1900, 8200, 2048), (1500, 8200, 2177), (60, 33001, 1153), (300, 777, 2049), (40, 1000, 1100)])
def test_random_values_are_near_on_the_whole(be, t, rows, cols):
    """Some rows and columns against 64 bits, element by element and in norm."""
    from test_gpu_f8 import rows_of

    rng = np.random.default_rng(t + cols)
    q, s = ref.random_matrix(rng, rows, cols, spread=3)
    w = be.upload_f8(q, s)
    x = rows_of(rng, t, cols, "bf16")
    d_x = be.to_device(x)
    r = np.unique(np.r_[0:4, t - 4:t, rng.integers(0, t, 60)])
    c = np.unique(np.r_[0:4, rows - 4:rows, rng.integers(0, rows, 300)])
    m = ref.TABLE[q[c]] * np.repeat(s.astype(np.float64)[c // 128], 128, 1)[:, :cols]
    for y_kind in ("f32", "bf16"):
        bt = np.uint16 if y_kind == "bf16" else np.float32
        d_y = be.to_device(np.full((t, rows), 7, bt))
        be.f8_matmul_device(w, d_x, t, d_y, x_type="bf16", y_type=y_kind)
        got = be.read(d_y, bt, (t, rows))[np.ix_(r, c)]
        got = (ref.from_bf16(got) if y_kind == "bf16" else got).astype(np.float64)
        want, tol = ref.matmul(ref.from_bf16(x[r]), m, y_kind == "bf16")
        assert np.all(np.abs(got - want) <= tol + ref.rounding(y_kind) * (np.abs(want) + tol) + 1e-40)
        # f32: random roundings of a sum of at most 2177 products and 18 blocks, sqrt(2195) * 2^-24.  bf16: its rounding,
        # even on +-2^-9 of a value's power of two, 2^-8 / sqrt(3) of the values at most, and 3.9e-5 of the fp8 cores
        bound = 47 * 2.0 ** -24 if y_kind == "f32" else 2.0 ** -8 / 3 ** 0.5 + 3.9e-5
        assert np.linalg.norm(got - want) <= bound * np.linalg.norm(want)
        be.free(d_y)
    be.free(d_x)
    be.free_weights(w)
