"""Attention over the cache at the longest lengths that a call takes: pages may stand in a table many times, so a few make a
sequence of 2^31 tokens."""
from __future__ import annotations

import math

import numpy as np
import pytest

import attn_ref as ref
import f8_ref
from test_gpu_attn_paged import be, bf16  # noqa: F401
from turboqwenfare_amd._lib import ERR_INVALID, HipError
from turboqwenfare_amd.backend import DeviceBuffer

pytestmark = pytest.mark.gpu

D = 64


@pytest.mark.parametrize("kind", ["bf16", "f8"])
@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("page", [16, 64])
def test_lengths_up_to_2_31(be, kind, odd, page):  # noqa: F811
    """All pages are page 0, whose keys have score 0, but the last one: there are 16 keys of 2^27 times their weight, without
    which the result is another.  odd: the last key's values are NaN, and only the last row sees it."""
    n = 2 ** 31 - page
    rng = np.random.default_rng(page)
    k = np.zeros((2, 1, page, D), np.float32)
    k[1, 0, -16:, :27] = 1.0
    one = {"bf16": 0x3F80, "f8": 0x38}[kind]
    kb = np.where(k == 1.0, one, 0).astype(np.uint16 if kind == "bf16" else np.uint8)
    if kind == "f8":
        vb, vs, v = ref.f8_cache(rng, k.shape)
        ks = np.ones(k.shape[:3], np.float32)
    else:
        vb, v = bf16(rng.standard_normal(k.shape))
    if odd:
        vb[1, 0, -1] = 0x7F if kind == "f8" else 0x7FC0
        v[1, 0, -1] = np.nan
    table = np.zeros(n // page, np.int32)
    table[-1] = 1
    q = bf16(np.ones((2, 1, D)))[0]
    bufs = [be.to_device(a) for a in (q, kb, vb, table, np.array([n], np.int32), np.zeros(2 * D, np.uint16), np.zeros(1, np.int32),
                                      *((ks, vs) if kind == "f8" else ()))]
    d_q, d_k, d_v, d_table, d_lens, d_y, d_status = bufs[:7]
    try:
        cache = be.kv_cache(d_k, d_v, 2, 1, page, D, kind, *bufs[7:])
        be.attn_paged_device(d_q, (1, 1, D), 1, 2, cache, d_table, len(table), d_lens, d_y, scale=math.log(2.0), d_status=d_status)
        got = f8_ref.from_bf16(be.read(d_y, np.uint16, (2, D))).astype(np.float64)
        status = be.read(d_status, np.int32, (1,))[0]
    finally:
        for b in bufs:
            be.free(b)
    weight = np.zeros((2, page))  # of page 0's and page 1's tokens, by the number of times that each is seen
    weight[0], weight[1] = len(table) - 1, 1.0
    weight[1, -16:] = 2.0 ** 27
    assert status == 0
    for row, seen in ((0, page - 1), (1, page)):
        w = weight.copy()
        w[1, seen:] = 0.0
        use = w > 0
        want, size = (w[use] / w.sum()) @ v[:, 0][use], (w[use] / w.sum()) @ np.abs(v[:, 0][use])
        # weights (2^-8 with their scales; 27 * ln 2 * log2 e in f32: 2^-18), y (2^-8), and 2^11 parts' sums in f32
        tol = size * (ref.BF16 + 2.0 ** -12) + (np.abs(want) + size * 2.0 ** -7) * ref.BF16
        if odd and row == 1:
            assert np.isnan(got[1]).all()
        else:
            assert (np.abs(got[row] - want) <= tol).all(), (row, got[row][:4], want[:4], tol[:4])


def test_most_keys_of_a_prompt(be):  # noqa: F811
    """Totals within a tile's 64 keys of 2^31 are refused: such a tile's end has no signed 32-bit number.  (The sequence itself
    has 5 keys; y lies in front of the keys, which only the total makes long.)"""
    whole = be.alloc(1 << 16)
    d_y, d_q, d_cu, d_k = (DeviceBuffer(whole.ptr + at, nbytes) for at, nbytes in ((0, 1 << 12), (1 << 12, 1 << 12), (1 << 13, 64), (1 << 14, 1 << 40)))
    be.write(whole, np.zeros(1 << 15, np.uint16))
    be.write(d_cu, np.array([0, 5], np.int32))
    be.write(d_k, np.full(5 * D, 0x3F80, np.uint16))
    try:
        for total in (2 ** 31 - 63, 2 ** 31 - 1):
            with pytest.raises(HipError) as e:
                be.attn_prompt_device(d_q, d_k, d_k, (1, 1, D), d_cu, d_cu, 1, 5, total, d_y)
            assert e.value.status == ERR_INVALID
        assert not be.read(d_y, np.uint16, (5 * D,)).any()
        be.attn_prompt_device(d_q, d_k, d_k, (1, 1, D), d_cu, d_cu, 1, 5, 2 ** 31 - 64, d_y)
        assert (be.read(d_y, np.uint16, (5 * D,)) == 0x3F80).all()
    finally:
        be.free(whole)
