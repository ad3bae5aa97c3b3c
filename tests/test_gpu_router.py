"""The batched router on the GPU: router_logits and route_tokens against their
definitions in 64 bits (f8_ref.py)."""
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


@pytest.fixture(scope="module")
def hip():
    from turboqwenfare_amd import backend

    return backend


def at(be, a, offset):
    """A device copy of `a` that begins `offset` bytes into its buffer; the whole buffer too."""
    a = np.ascontiguousarray(a)
    whole = be.to_device(np.concatenate([np.zeros(offset, np.uint8), a.reshape(-1).view(np.uint8), np.zeros(64, np.uint8)]))
    return be.view(whole, offset, a.nbytes), whole


# ---- logits ---------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("t,n,hidden,offset", [
    (1, 256, 2048, 0), (3, 7, 33, 4), (8, 256, 2048, 0), (8, 1, 1, 0), (9, 256, 2048, 0), (9, 1, 5, 4), (33, 60, 1000, 0),
    (37, 17, 71, 4), (64, 256, 256, 0), (513, 256, 264, 0), (530, 65, 333, 4), (577, 1000, 40, 0)])
def test_logits(be, kind, t, n, hidden, offset):
    rng = np.random.default_rng(t * 1000 + n + hidden)
    x = (rng.standard_normal((t, hidden)) * np.exp2(rng.integers(-12, 5, (1, hidden)))).astype(np.float32)
    r = (rng.standard_normal((n, hidden)) * hidden ** -0.5).astype(np.float32)
    bits = ref.to_bf16(x) if kind == "bf16" else x
    xv = (ref.from_bf16(bits) if kind == "bf16" else x).astype(np.float64)
    w = be.upload_f32(r)
    d_x, whole = at(be, bits, offset if kind == "f32" else offset // 2)
    guard = np.full(t * n + 16, 7.0, np.float32)
    d_l = be.to_device(guard)
    be.router_logits_device(w, d_x, t, n, hidden, d_l, x_type=kind)
    got = be.read(d_l, np.float32, guard.shape)
    assert np.array_equal(got[t * n:], guard[t * n:])
    got = got[:t * n].reshape(t, n)
    want, mag = xv @ r.astype(np.float64).T, np.abs(xv) @ np.abs(r.astype(np.float64)).T
    # few rows: one rounding of a 64-bit sum; else f32 sums of at most `hidden` exact parts (three or six per product),
    # and 3 * 2^-24 of an f32 product is left out
    tol = 2.0 ** -24 * np.abs(want) + 2.0 ** -45 * mag if t <= 8 else (hidden + 24) * 2.0 ** -23 * mag
    assert np.all(np.abs(got - want) <= tol + 1e-37)
    for b in (whole, d_l):
        be.free(b)
    be.free_tensor(w)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("hidden", [32, 256, 320, 327])
def test_logits_of_every_tile_size(be, kind, hidden):
    """Row and expert counts on both sides of each change of tile: near 64 bits, and bit by bit the same number for a
    row and an expert whatever stands beside them (the order of the sum does not depend on the tile)."""
    rng = np.random.default_rng(hidden)
    t, n = 4096, 259
    x, r = rng.standard_normal((t, hidden)).astype(np.float32), rng.standard_normal((n, hidden)).astype(np.float32)
    bits = ref.to_bf16(x) if kind == "bf16" else x
    xv = (ref.from_bf16(bits) if kind == "bf16" else x).astype(np.float64)
    want, mag = xv @ r.astype(np.float64).T, np.abs(xv) @ np.abs(r.astype(np.float64)).T
    tol = (hidden + 24) * 2.0 ** -23 * mag  # as above
    d_x = be.to_device(bits)
    whole = None
    for rows, experts in ((t, n), (t, 17), (1969, 259), (1921, 256), (1025, 256), (1000, 256), (513, 256), (481, 259), (9, 259), (t, 1)):
        w = be.upload_f32(r[:experts])
        guard = np.full(rows * experts + 16, 7.0, np.float32)
        d_l = be.to_device(guard)
        be.router_logits_device(w, d_x, rows, experts, hidden, d_l, x_type=kind)
        got = be.read(d_l, np.float32, guard.shape)
        assert np.array_equal(got[rows * experts:], guard[rows * experts:])
        got = got[:rows * experts].reshape(rows, experts)
        assert np.all(np.abs(got - want[:rows, :experts]) <= tol[:rows, :experts])
        whole = got if whole is None else whole
        assert np.array_equal(got, whole[:rows, :experts])
        be.free(d_l)
        be.free_tensor(w)
    be.free(d_x)


def test_logits_are_near_f32(be):
    """Far from the worst case, both paths are as near to 64 bits as a rounding or two of an f32 sum."""
    rng = np.random.default_rng(5)
    x, r = rng.standard_normal((600, 2048)).astype(np.float32), (rng.standard_normal((256, 2048)) / 45).astype(np.float32)
    w = be.upload_f32(r)
    want = x.astype(np.float64) @ r.astype(np.float64).T
    for rows in (8, 100, 600):
        got = be.router_logits(w, x[:rows])
        err = np.linalg.norm(got - want[:rows]) / np.linalg.norm(want[:rows])
        # random errors of 2^-24 a step in a sum of 2048 add as the square root: 45 * 2^-24 = 2.7e-6
        assert err < 2.7e-6, (rows, err)
    be.free_tensor(w)


def test_rows_of_logits_do_not_see_each_other(be):
    rng = np.random.default_rng(6)
    for t in (8, 40, 600):
        x, r = rng.standard_normal((t, 200)).astype(np.float32), rng.standard_normal((32, 200)).astype(np.float32)
        w = be.upload_f32(r)
        clean = be.router_logits(w, x)
        x[t // 2, 17] = np.nan
        x[t // 3, 0] = np.inf
        got = be.router_logits(w, x)
        rest = np.ones(t, bool)
        rest[[t // 2, t // 3]] = False
        assert np.isnan(got[t // 2]).all() and not np.isfinite(got[t // 3]).any()
        assert np.array_equal(got[rest], clean[rest])
        be.free_tensor(w)


# ---- routes ----------------------------------------------------------------------------
OPTIONS = [
    dict(), dict(renormalise=False, scale=1.5), dict(score="sigmoid"), dict(score="sigmoid", renormalise=False, scale=-2.5),
    dict(n_groups=8, top_groups=4, group_best=2, score="sigmoid", scale=2.5), dict(n_groups=4, top_groups=1),
    dict(n_groups=4, top_groups=4, group_best=2)]


def check(be, lg, top_k, bias=None, **o):
    ids, w = be.route_tokens(lg, top_k, bias, **o)
    want, p, failed = ref.route(lg, top_k, bias=bias, **o)
    assert not failed
    assert np.array_equal(ids, want)
    # a rounding of a 64-bit number
    assert np.all(np.abs(w - p) <= 2.0 ** -24 * np.abs(p) * (1 + 1e-6) + 1e-45)
    return ids, w


@pytest.mark.parametrize("o", OPTIONS)
@pytest.mark.parametrize("t,n,top_k", [(1, 256, 8), (5, 8, 2), (131, 256, 8), (67, 512, 16), (33, 1024, 3), (3, 64, 16)])
def test_routes(be, t, n, top_k, o):
    if top_k > o.get("top_groups", 1) * n // o.get("n_groups", 1):
        pytest.skip("more routes than experts kept")
    rng = np.random.default_rng(t + n)
    lg = (rng.standard_normal((t, n)) * 2).astype(np.float32)
    check(be, lg, top_k, **o)
    check(be, lg, top_k, bias=(rng.standard_normal(n) * 0.1).astype(np.float32), **o)


@pytest.mark.parametrize("n,groups,kept,top_k", [(1, 1, 1, 1), (7, 1, 1, 7), (65, 5, 2, 16), (99, 3, 2, 11), (1023, 33, 4, 16), (1020, 17, 3, 16),
                                                 (64, 64, 9, 9), (1024, 64, 64, 16), (130, 2, 1, 1), (1000, 1, 1, 16)])
def test_sizes_that_fit_no_wavefront(be, n, groups, kept, top_k):
    rng = np.random.default_rng(n)
    lg = rng.standard_normal((19, n)).astype(np.float32)
    for score in ("softmax", "sigmoid"):
        check(be, lg, top_k, score=score, n_groups=groups, top_groups=kept, group_best=2)


def test_ties_go_to_the_lowest(be):
    rng = np.random.default_rng(3)
    lg = rng.integers(-1, 2, (200, 256)).astype(np.float32)  # a third of the experts tie
    for o in OPTIONS:
        check(be, lg, 8, **o)
    check(be, np.zeros((4, 300), np.float32), 16)
    check(be, np.zeros((4, 320), np.float32), 16, n_groups=5, top_groups=2, group_best=1)
    # scores that are one in f32 and two in f64
    one = np.zeros((1, 64), np.float32)
    one[0, 40], one[0, 9] = 30.0, 29.0
    ids, _ = check(be, one, 2, score="sigmoid")
    assert ids.tolist() == [[40, 9]]


def test_masked_experts(be):
    rng = np.random.default_rng(4)
    lg = rng.standard_normal((64, 256)).astype(np.float32)
    lg[rng.random(lg.shape) < 0.3] = -np.inf
    lg[3], lg[17, 5:] = -np.inf, -np.inf       # nothing left; five left
    lg[20] = np.finfo(np.float32).min          # the lowest value is a value
    lg[21, 1:] = -np.inf
    bias = rng.standard_normal(256).astype(np.float32)
    bias[50:60] = -np.inf
    for o in OPTIONS:
        for b in (None, bias):
            ids, w = check(be, lg, 8, bias=b, **o)
            assert (ids[3] == ref.NONE).all() and (w[3] == 0).all()


def test_extreme_logits(be):
    lg = np.zeros((6, 128), np.float32)
    lg[0, 5], lg[1, 7] = np.finfo(np.float32).max, np.finfo(np.float32).min
    lg[2], lg[3] = -200.0, np.finfo(np.float32).min
    lg[4, :64], lg[5, ::2] = 800.0, -800.0
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            check(be, lg, 8, score=score, renormalise=renorm)


def test_rows_that_fail_alone(be, hip):
    rng = np.random.default_rng(8)
    t, n = 40, 256
    lg = rng.standard_normal((t, n)).astype(np.float32)
    lg[7, 200], lg[30, 0], lg[31, 9] = np.nan, np.inf, -np.inf
    d = [be.to_device(a) for a in (lg, np.zeros((t, 8), np.uint16), np.zeros((t, 8), np.float32), np.zeros(1, np.int32))]
    be.route_tokens_device(d[0], t, n, 8, d[1], d[2], d_status=d[3])
    ids, w, st = be.read(d[1], np.uint16, (t, 8)), be.read(d[2], np.float32, (t, 8)), be.read(d[3], np.int32, (1,))
    want, p, failed = ref.route(lg, 8)
    assert failed == [7, 30] and st[0] == 4
    assert np.array_equal(ids, want) and np.allclose(w, p, rtol=2.0 ** -23, atol=0)
    with pytest.raises(hip.HipError):
        be.route_tokens(lg, 8)
    # a bias that is no number takes every row down, unless its expert is masked
    bias = np.zeros(n, np.float32)
    bias[9] = np.nan
    d_b = be.to_device(bias)
    be.write(d[3], np.zeros(1, np.int32))
    be.route_tokens_device(d[0], t, n, 8, d[1], d[2], d_bias=d_b, d_status=d[3])
    ids = be.read(d[1], np.uint16, (t, 8))
    assert (ids[np.arange(t) != 31] == ref.NONE).all() and (ids[31] != ref.NONE).all()
    for b in (*d, d_b):
        be.free(b)


def test_bf16_logits_and_what_lies_behind(be):
    rng = np.random.default_rng(9)
    t, n, k = 21, 100, 5
    bits = ref.to_bf16(rng.standard_normal((t, n)).astype(np.float32))
    d_l, whole = at(be, bits, 2)
    d_i, d_w = be.to_device(np.full(t * k + 9, 1234, np.uint16)), be.to_device(np.full(t * k + 9, 5.0, np.float32))
    be.route_tokens_device(d_l, t, n, k, d_i, d_w, logits_type="bf16")
    ids, w = be.read(d_i, np.uint16, (t * k + 9,)), be.read(d_w, np.float32, (t * k + 9,))
    want, p, _ = ref.route(ref.from_bf16(bits), k)
    assert np.array_equal(ids[:t * k].reshape(t, k), want) and (ids[t * k:] == 1234).all()
    assert np.allclose(w[:t * k].reshape(t, k), p, rtol=2.0 ** -23, atol=0) and (w[t * k:] == 5.0).all()
    for b in (whole, d_i, d_w):
        be.free(b)


def test_same_ids_as_the_layer_kernels(be):
    """Softmax, top-8, renormalised: the ids that the router of an MoE layer takes from the same logits."""
    import cpu_oracle as orc

    rng = np.random.default_rng(10)
    lg = (rng.standard_normal((50, 256)) * 2).astype(np.float32)
    ids, w = be.route_tokens(lg, 8)
    for r in range(50):
        oid, ow = orc.router_from_logits(lg[r])
        assert np.array_equal(ids[r], oid)
        # the oracle's are sequential f32 sums of 256 and 8
        assert np.allclose(w[r], ow, rtol=(256 + 16) * 2.0 ** -24, atol=0)


def test_refusals(be, hip):
    from turboqwenfare_amd import _lib

    d = be.alloc(1 << 16)
    i, w = be.alloc(1 << 12), be.alloc(1 << 12)
    ok = dict(t=4, n_experts=16, top_k=2)

    def call(**o):
        o = {**ok, **o}
        be.route_tokens_device(d, o.pop("t"), o.pop("n_experts"), o.pop("top_k"), o.pop("d_ids", i), o.pop("d_w", w), **o)

    call()
    for bad in (dict(t=0), dict(n_experts=0, top_k=1), dict(top_k=0), dict(top_k=17, n_experts=32), dict(n_groups=3), dict(n_groups=0),
                dict(n_groups=4, top_groups=5), dict(n_groups=4, top_groups=0), dict(group_best=3), dict(group_best=0), dict(scale=float("nan")),
                dict(n_groups=8, top_groups=1, top_k=3), dict(t=1, n_experts=2048), dict(d_ids=be.view(i, 1, 100)), dict(d_w=be.view(w, 2, 100)),
                dict(d_ids=be.view(d, 0, 1000)), dict(t=65537, n_experts=1, top_k=1, d_ids=hip.DeviceBuffer(i.ptr, 1 << 30), d_w=hip.DeviceBuffer(w.ptr, 1 << 30))):
        if "t" in bad and bad["t"] > 65536:
            big = hip.DeviceBuffer(d.ptr, 1 << 30)
            with pytest.raises(hip.HipError) as e:
                be.route_tokens_device(big, 65537, 1, 1, bad["d_ids"], bad["d_w"])
        else:
            with pytest.raises(hip.HipError) as e:
                call(**bad)
        assert e.value.status == _lib.ERR_INVALID, bad
    for bad in (dict(t=5000), dict(score="top"), dict(logits_type="f16")):
        with pytest.raises(ValueError):
            call(**bad)
    r = be.upload_f32(np.zeros(64, np.float32))
    be.router_logits_device(r, d, 2, 4, 16, w)
    for args in ((r, d, 2, 4, 15, w), (r, d, 0, 4, 16, w), (r, d, 2, 0, 16, w), (r, d, 2, 4, 16, be.view(d, 4, 1000)), (r, be.view(d, 2, 1000), 2, 4, 16, w)):
        with pytest.raises(hip.HipError) as e:
            be.router_logits_device(*args)
        assert e.value.status == _lib.ERR_INVALID
    be.free_tensor(r)
    for b in (d, i, w):
        be.free(b)
