"""F8 experts whose outputs pass what f32 holds, or come near zero."""
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


@pytest.mark.parametrize("y_kind", ["f32", "bf16"])
@pytest.mark.parametrize("n,t,k", [(1, 3, 1), (1, 40, 1), (1, 400, 1), (130, 2000, 1), (130, 4096, 2)])
def test_outputs_at_both_ends_of_f32(be, n, t, k, y_kind):
    """Experts whose h has one value that is not zero, times what their down matrix gives: a column that passes the
    largest f32 beside columns of zeros, and columns of 2^-101 and 2^-115.  Slots by themselves and tiles of every size."""
    H = 384
    one = int(np.flatnonzero(ref.TABLE == 1.0)[0])
    gate, up, down = np.zeros((128, H), np.uint8), np.zeros((128, H), np.uint8), np.zeros((H, 128), np.uint8)
    gate[0, 0] = up[0, 0] = one
    down[[0, 290], 0], down[[130, 200], 0] = (int(np.flatnonzero(ref.TABLE == v)[0]) for v in (448.0, 2.0 ** -6))
    # x[0] = 448, so its scale is 1; silu(448) is 448; h = 448^2 = 448 * 448, so its scale is 448 and its value 448
    s = np.ones((1, 3), np.float32)
    down_s = np.array([[2.0 ** 118], [2.0 ** -125], [2.0 ** -126]], np.float32)
    h = [[be.upload_f8(gate, s)], [be.upload_f8(up, s)], [be.upload_f8(down, down_s)]]
    ex = be.prepare_f8_experts(*([m] * n for (m,) in h))
    x = np.zeros((t, H), np.float32)
    x[:, 0] = 448
    bt = np.uint16 if y_kind == "bf16" else np.float32
    d = [be.to_device(a) for a in (x, (np.arange(t * k) % n).reshape(t, k).astype(np.uint16), np.full((t, k), 1 / k, np.float32), np.full((t, H), 7, bt))]
    be.f8_experts_device(ex, d[0], t, d[1], d[2], k, d[3], y_type=y_kind)
    got = be.read(d[3], bt, (t, H))
    got = (ref.from_bf16(got) if y_kind == "bf16" else got).astype(np.float64)
    want = np.zeros(H)
    # 448^3 = 343 * 2^18: nine bits, so bf16 rounds it, to even
    want[[0, 130, 200, 290]] = np.inf, 448.0 ** 2 * 2.0 ** -131, 448.0 ** 2 * 2.0 ** -131, 448.0 ** 3 * 2.0 ** -126
    if y_kind == "bf16":
        want = ref.from_bf16(ref.to_bf16(want.astype(np.float32))).astype(np.float64)
    assert np.array_equal(got, np.broadcast_to(want, (t, H))), got[0, [0, 1, 130, 131, 290]]
    for b in d:
        be.free(b)
    be.free_f8_experts(ex)
    for g in h:
        for m in g:
            be.free_weights(m)
