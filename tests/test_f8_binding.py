"""What the host forms of the F8 calls make of other integer types, and what they refuse (on the CPU)."""
from __future__ import annotations

import numpy as np
import pytest

import f8_ref as ref
from turboqwenfare_amd import backend


class Taken(Exception):
    pass


@pytest.fixture
def be():
    """The binding without a device; a call that reaches the library raises Taken with what it was given."""
    class Lib:
        def __getattr__(self, name):
            def call(*args):
                raise Taken(name, args)
            return call

    b = backend.HipBackend.__new__(backend.HipBackend)
    b.lib, b.ctx = Lib(), None

    def to_device(a):
        raise Taken("to_device", a)
    b.to_device = to_device
    return b


def test_bytes_are_bytes(be):
    """Values given for bytes, or numbers that no byte holds, would be cut to other numbers."""
    s = np.ones((1, 1), np.float32)
    for q in (np.zeros((2, 3), np.uint8), np.full((2, 3), -1, np.int8), np.full((2, 3), 255, np.int64)):
        with pytest.raises(Taken):
            be.upload_f8(q, s)
    for q in (np.full((2, 3), 0.5, np.float32), np.full((2, 3), 256), np.full((2, 3), -129), [[1.0, 2.0]]):
        with pytest.raises(ValueError):
            be.upload_f8(q, s)


def test_ids_are_not_cut(be):
    """-1 is the empty slot, as 0xFFFF is; an id of 65537 is no expert 1."""
    ex = backend.F8Experts(1, 4, 64, 32, [])
    x, w = np.zeros((2, 64), np.float32), np.zeros((2, 2), np.float32)
    for ids in (np.zeros((2, 2), np.uint16), np.full((2, 2), -1), np.full((2, 2), ref.NONE, np.int32)):
        with pytest.raises(Taken):
            be.f8_experts(ex, x, ids, w)
    for ids in (np.full((2, 2), 65537), np.full((2, 2), -2), np.full((2, 2), 1.0)):
        with pytest.raises(ValueError):
            be.f8_experts(ex, x, ids, w)
