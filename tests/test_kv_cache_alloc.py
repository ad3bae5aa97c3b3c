"""Buffers of a cache that cannot be made are given back (on the CPU)."""
from __future__ import annotations

import pytest

from turboqwenfare_amd import backend
from turboqwenfare_amd._lib import ERR_NOMEM, HipError
from turboqwenfare_amd.backend import DeviceBuffer


@pytest.fixture
def be():
    b = backend.HipBackend.__new__(backend.HipBackend)
    b.live, b.left = {}, 100

    def alloc(nbytes):
        if not b.left:
            raise HipError(ERR_NOMEM, "no memory")
        b.left -= 1
        b.live[b.left] = nbytes
        return DeviceBuffer(b.left, nbytes)

    b.alloc, b.free = alloc, lambda buf: b.live.pop(buf.ptr)
    return b


@pytest.mark.parametrize("kind", ["fp8", "f32", ""])
def test_unknown_types(be, kind):
    with pytest.raises(ValueError):
        be.alloc_kv_cache(8, 2, 16, 64, kind)
    assert be.live == {}


@pytest.mark.parametrize("kind, n", [("bf16", 2), ("f8", 4)])
def test_no_memory(be, kind, n):
    for left in range(n):
        be.left = left
        with pytest.raises(HipError):
            be.alloc_kv_cache(8, 2, 16, 64, kind)
        assert be.live == {}
    be.left = n
    c = be.alloc_kv_cache(8, 2, 16, 64, kind)
    assert sorted(be.live.values()) == sorted([8 * 2 * 16 * 64 * (2 if kind == "bf16" else 1)] * 2 + ([8 * 2 * 16 * 4] * 2 if kind == "f8" else []))
    be.free_kv_cache(c)
    assert be.live == {}
