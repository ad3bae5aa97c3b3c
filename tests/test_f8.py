"""CPU checks of the e4m3 format's oracle and of what the binding refuses
before it reaches the library."""
from __future__ import annotations

import numpy as np
import pytest

import f8_ref as ref
from turboqwenfare_amd import _lib, backend


def test_the_table_is_e4m3():
    import torch

    b = torch.arange(256, dtype=torch.uint8)
    assert np.array_equal(ref.TABLE, b.view(torch.float8_e4m3fn).double().numpy(), equal_nan=True)


def test_rounding_is_e4m3s():
    import torch

    t = ref.TABLE[:127]
    mid = (t[1:] + t[:-1]) / 2
    z = np.concatenate([t, mid, np.nextafter(mid, 0), np.nextafter(mid, 1e9), np.random.default_rng(0).standard_normal(20000) * 50]).astype(np.float32)
    z = z[np.abs(z) <= 448]
    for v in (z, -z):
        assert np.array_equal(ref.round_e4m3(v), torch.from_numpy(v).to(torch.float8_e4m3fn).double().numpy())


def test_quantised_rows():
    x = np.zeros((3, 200), np.float32)
    x[0] = np.linspace(-3, 5, 200)
    x[1, 130] = 2.0 ** -101
    x[2, 7] = np.finfo(np.float32).max
    q, s, _ = ref.quantize(x)
    assert np.abs(q[0, :128]).max() == 448 and np.abs(q[0, 128:]).max() == 448
    assert np.all(np.abs(q[0] * s[0] - x[0]) <= 2.0 ** -4 * np.abs(x[0]) + s[0] * 2.0 ** -10)
    assert (q[1] == 0).all() and q[2, 7] == 448 and np.isfinite(s).all()


def test_routes_by_hand():
    lg = np.log(np.array([[0.1, 0.4, 0.3, 0.2]]))
    ids, w, failed = ref.route(lg, 2)
    assert ids.tolist() == [[1, 2]] and np.allclose(w, [[4 / 7, 3 / 7]]) and not failed
    ids, w, _ = ref.route(lg, 2, n_groups=2, top_groups=1, renormalise=False, bias=[0.5, 0, 0, 0])
    assert ids.tolist() == [[0, 1]] and np.allclose(w, [[0.1, 0.4]])
    ids, w, _ = ref.route([[-np.inf, 0.0, -np.inf]], 2, score="sigmoid")
    assert ids.tolist() == [[1, ref.NONE]] and w.tolist() == [[1.0, 0.0]]


@pytest.mark.parametrize("rows,cols,tiles,blocks", [(1, 1, 4, 1), (128, 128, 4, 1), (129, 257, 8, 3), (151936, 2048, 4748, 16)])
def test_bytes_of_an_upload(rows, cols, tiles, blocks):
    need = tiles * blocks * 4096 + tiles // 4 * blocks * 4
    assert backend.HipBackend.f8_weights_bytes_for(rows, cols) == -(-need // 256) * 256


def test_shapes_that_do_not_fit():
    for rows, cols in ((0, 1), (1, 0), ((1 << 24) + 1, 1), (1, 65537)):
        assert backend.HipBackend.f8_weights_bytes_for(rows, cols) == 0


@pytest.fixture
def be(monkeypatch):
    """The binding without a device: a call that reaches the library fails the test."""
    class Lib:
        def __getattr__(self, name):
            raise AssertionError(f"{name} was called")

    b = backend.HipBackend.__new__(backend.HipBackend)
    b.lib, b.ctx = Lib(), None
    return b


def test_the_binding_refuses(be):
    w, ex = backend.F8Weights(1, 32, 256), backend.F8Experts(1, 4, 64, 32, [])
    buf = lambda n: backend.DeviceBuffer(256, n)  # noqa: E731
    r = backend.F32Tensor(1, 64)
    for call in (
            lambda: be.upload_f8(np.zeros((4, 4), np.uint8), np.ones((2, 1), np.float32)),
            lambda: be.upload_f8(np.zeros(4, np.uint8), np.ones((1, 1), np.float32)),
            lambda: be.upload_f8_device(buf(15), buf(4), 4, 4),
            lambda: be.upload_f8_device(buf(16), buf(3), 4, 4),
            lambda: be.f8_matmul_device(w, buf(4 * 256), 2, buf(1 << 20)),
            lambda: be.f8_matmul_device(w, buf(1 << 20), 2, buf(4 * 32)),
            lambda: be.f8_matmul_device(w, buf(1 << 20), 2, buf(1 << 20), x_type="f64"),
            lambda: be.f8_matmul(w, np.zeros((2, 255), np.float32)),
            lambda: be.prepare_f8_experts([], [], []),
            lambda: be.prepare_f8_experts([w], [w, w], [w]),
            lambda: be.f8_experts_device(ex, buf(1 << 20), 4, buf(15), buf(1 << 20), 2, buf(1 << 20)),
            lambda: be.f8_experts_device(ex, buf(1 << 20), 4, buf(16), buf(31), 2, buf(1 << 20)),
            lambda: be.f8_experts_device(ex, buf(1 << 20), 4, buf(16), buf(32), 2, buf(4 * 64 * 2), y_type="f32"),
            lambda: be.f8_experts(ex, np.zeros((2, 64), np.float32), np.zeros((2, 2), np.uint16), np.zeros((2, 3), np.float32)),
            lambda: be.router_logits_device(r, buf(127), 2, 4, 16, buf(1 << 20)),
            lambda: be.router_logits(r, np.zeros((2, 15), np.float32)),
            lambda: be.route_tokens_device(buf(1 << 20), 2, 16, 2, buf(8), buf(15)),
            lambda: be.route_tokens_device(buf(1 << 20), 2, 16, 2, buf(8), buf(16), d_bias=buf(63)),
            lambda: be.route_tokens_device(buf(1 << 20), 2, 16, 2, buf(8), buf(16), score="max"),
            lambda: be.route_tokens(np.zeros((2, 16), np.float32), 2, bias=np.zeros(15, np.float32))):
        with pytest.raises(ValueError):
            call()


def test_options_are_laid_out_as_in_the_header():
    import ctypes

    assert ctypes.sizeof(_lib.RouteOptions) == 28
    assert [f[0] for f in _lib.RouteOptions._fields_] == ["score", "top_k", "n_groups", "top_groups", "group_best", "renormalise", "scale"]
