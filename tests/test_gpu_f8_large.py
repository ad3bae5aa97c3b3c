"""F8 calls whose buffers pass 2^31 and 2^32 bytes: the rows, h and the matrix.  Integers, so that the sums are exact; some
rows and columns are looked at."""
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


def repeated(be, a, rows):
    """A device buffer of `rows` rows, a's over and over."""
    whole, one = be.alloc(rows * a[0].nbytes), be.to_device(a)
    for at in range(0, rows, len(a)):
        n = min(len(a), rows - at) * a[0].nbytes
        be.copy_device(be.view(whole, at * a[0].nbytes, n), one, n)
    be.synchronize()
    be.free(one)
    return whole


def some_rows(be, d, pick, cols, dtype):
    size = np.dtype(dtype).itemsize * cols
    return np.stack([be.read(be.view(d, int(r) * size, size), dtype, (cols,)) for r in pick])


CODES = np.array([int(np.flatnonzero(ref.TABLE == v)[0]) for v in range(-4, 5)], np.uint8)
TYPES = {"f32": np.float32, "bf16": np.uint16}


@pytest.mark.parametrize("rows,y_kind", [(300, "bf16"), (1000, "bf16"), (140, "f32")])
def test_rows_of_2_to_the_32_bytes(be, rows, y_kind):
    """65535 rows of 65536 columns, quantised to 2^32 - 65536 bytes: tiles of 96 and 256 rows, and of 64 for f32."""
    t, cols, own = 65535, 65536, 2003
    rng = np.random.default_rng(rows)
    x = rng.integers(-7, 8, (own, cols), dtype=np.int8)
    x[:, ::128] = 7  # each block's largest, so that its scale is 2^-6
    table = ref.to_bf16(np.arange(-7, 8, dtype=np.float32))
    d_x = repeated(be, table[x + 7], t)
    at = rng.integers(0, 9, (rows, cols), dtype=np.int8)
    w = be.upload_f8(CODES[at], np.ones((-(-rows // 128), cols // 128), np.float32))
    d_y = be.alloc(t * rows * np.dtype(TYPES[y_kind]).itemsize)
    be.f8_matmul_device(w, d_x, t, d_y, x_type="bf16", y_type=y_kind)
    pick = np.r_[0:20, 32750:32780, t - 20:t]
    got = some_rows(be, d_y, pick, rows, TYPES[y_kind])
    # sums of integers up to 28 * 65536 < 2^24: exact in f32, in any order
    want = x[pick % own].astype(np.float32) @ (at.astype(np.float32) - 4).T
    assert np.array_equal(got, ref.to_bf16(want) if y_kind == "bf16" else want)
    be.free_weights(w)
    for b in (d_x, d_y):
        be.free(b)


def test_a_matrix_of_2_to_the_33_bytes(be):
    """131100 rows of 65536 columns: the weight stream (as many rows as fit its LDS), and tiles."""
    rows, cols, own = 131100, 65536, 2003
    rng = np.random.default_rng(1)
    at = rng.integers(0, 9, (own, cols), dtype=np.int8)
    d_q, d_s = repeated(be, CODES[at], rows), be.to_device(np.ones((-(-rows // 128), cols // 128), np.float32))
    w = be.upload_f8_device(d_q, d_s, rows, cols)
    be.free(d_q)
    x = rng.integers(-7, 8, (70, cols)).astype(np.float32)
    x[:, ::128] = 7
    want = np.tile(x @ (at.astype(np.float32) - 4).T, (1, -(-rows // own)))[:, :rows]
    d_x = be.to_device(ref.to_bf16(x))
    for t in (1, 12, 20, 70):
        for y_kind, dtype in TYPES.items():
            d_y = be.to_device(np.full((t, rows), 7, dtype))
            be.f8_matmul_device(w, d_x, t, d_y, x_type="bf16", y_type=y_kind)
            got = be.read(d_y, dtype, (t, rows))
            assert np.array_equal(got, ref.to_bf16(want[:t]) if y_kind == "bf16" else want[:t]), (t, y_kind)
            be.free(d_y)
    be.free_weights(w)
    for b in (d_s, d_x):
        be.free(b)


def test_h_of_2_to_the_32_bytes(be):
    """4096 tokens of 16 slots through experts of width 65408: h takes 2^32 - 2^23 bytes."""
    from test_gpu_f8 import Layer, rows_of, values_of

    n, hidden, width, t, k = 2, 16, 65408, 4096, 16
    layer = Layer(be, n, hidden, width, 2)
    rng = np.random.default_rng(0)
    bits = rows_of(rng, t, hidden, "f32")
    ids = rng.integers(0, n, (t, k)).astype(np.uint16)
    ids[rng.random((t, k)) < 0.1] = ref.NONE
    w = np.where(ids == ref.NONE, np.nan, rng.random((t, k)) / k).astype(np.float32)
    pick = np.r_[0:3, 2047, 2049, t - 2:t]
    for y_kind in ("f32", "bf16"):
        got, st = layer.run(bits, "f32", ids, w, y_kind)
        assert st == 0
        want, tol = ref.experts(bits[pick], ids[pick], w[pick], layer.mats, y_kind == "bf16", y_kind)
        # and 2^-11 of a term that waits as f16: the magnitudes of the terms, which are those of a single expert's y
        part = sum(np.abs(ref.experts(bits[pick], ids[pick][:, i:i + 1], w[pick][:, i:i + 1], layer.mats, False, "f32")[0]) for i in range(k))
        tol = tol + (2.0 ** -11 * part if y_kind == "bf16" else 0)
        assert np.all(np.abs(values_of(got, y_kind)[pick] - want) <= tol + 1e-35)
    layer.close()
