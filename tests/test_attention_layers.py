"""Attention layers on the CPU: arguments, what is given back, and the loop's handling of prompts (no GPU)."""
from __future__ import annotations

import numpy as np
import pytest

from turboqwenfare_amd.attention import AttentionLayers, f8_synthetic
from turboqwenfare_amd.backend import DeviceBuffer, KvCache
from turboqwenfare_amd.mtp_loop import MtpLoop


class Recorder:
    """Stands for the backend: handles are numbers, calls are kept, allocation `fail_at` fails."""

    def __init__(self, fail_at=None):
        self.n, self.live, self.calls, self.fail_at = 0, {}, [], fail_at

    def _new(self, nbytes=0):
        self.n += 1
        if self.n == self.fail_at:
            raise RuntimeError("no memory")
        self.live[4096 * self.n] = nbytes
        return 4096 * self.n

    def _gone(self, ptr):
        del self.live[ptr]

    def alloc(self, nbytes):
        return DeviceBuffer(self._new(nbytes), nbytes)

    def to_device(self, a):
        return self.alloc(a.nbytes)

    def prepare_rope(self, f):
        return self._new()

    def upload_f32(self, a):
        return self._new()

    def upload_f8(self, q, s):
        return self._new()

    free_rope = free_tensor = free_weights = _gone

    def free(self, b):
        self._gone(b.ptr)

    def alloc_kv_cache(self, pages, nk, page, d, kind):
        return KvCache(self.alloc(2 * pages * nk * page * d), self.alloc(2 * pages * nk * page * d), pages, nk, page, d, kind)

    def free_kv_cache(self, c):
        self.free(c.d_k), self.free(c.d_v)

    @staticmethod
    def view(buf, offset, nbytes):
        assert offset >= 0 and offset + nbytes <= buf.nbytes
        return DeviceBuffer(buf.ptr + offset, nbytes)

    def __getattr__(self, name):
        if name.startswith("_") or not name.endswith("_device"):
            raise AttributeError(name)
        return lambda *args, **kw: self.calls.append((name, args, kw))


SMALL = dict(heads=(4, 2, 64), rotary=32, max_tokens=40, page=16)


def test_all_is_given_back_also_after_a_failure():
    be = Recorder()
    AttentionLayers(be, 2, **SMALL).free()
    assert not be.live
    for i in range(1, be.n + 1):
        other = Recorder(fail_at=i)
        with pytest.raises(RuntimeError):
            AttentionLayers(other, 2, **SMALL)
        # a cache's own buffers are its maker's to give back
        assert len(other.live) <= 1


def test_arguments():
    for bad in (dict(rotary=31), dict(rotary=66), dict(rotary=-2), dict(max_tokens=0)):
        with pytest.raises(ValueError):
            AttentionLayers(Recorder(), 1, **{**SMALL, **bad})
    with pytest.raises(ValueError):
        AttentionLayers(Recorder(), 0, **SMALL)


def test_which_attention_runs_and_at_what_positions():
    be = Recorder()
    layers = AttentionLayers(be, 1, **SMALL)
    x = DeviceBuffer(1 << 40, 1 << 30)
    for t, at, name in ((9, 0, "attn_prompt_device"), (40, 0, "attn_prompt_device"), (1, 0, "attn_paged_device"), (8, 0, "attn_paged_device"),
                        (8, 32, "attn_paged_device"), (1, 39, "attn_paged_device")):
        be.calls.clear()
        layers.forward(0, x, t, at)
        names = [c[0] for c in be.calls]
        assert [n for n in names if n.startswith("attn")] == [name]
        rope = next(c for c in be.calls if c[0] == "qk_rope_device")
        assert rope[1][3] == t and rope[1][5].ptr == layers.d_count.ptr + 4 * at and rope[2]["d_slots"].ptr == layers.d_slots.ptr + 4 * at
        assert (rope[2]["d_k_out"] is not None) == (name == "attn_prompt_device")
        if name == "attn_paged_device":
            call = next(c for c in be.calls if c[0] == name)
            assert call[1][3] == t and call[1][7].ptr == layers.d_count.ptr + 4 * (at + t)
    for t, at in ((0, 0), (41, 0), (1, 40), (2, 39), (9, 1), (1, -1)):
        with pytest.raises(ValueError):
            layers.forward(0, x, t, at)


def test_synthetic_matrices_have_rows_of_unit_gain():
    q, s = f8_synthetic(256, 512, 1)
    assert not ((q & 127) == 127).any() and s.shape == (2, 4) and s.dtype == np.float32
    m = q & 127
    e, f = m >> 3, (m & 7).astype(np.float64)
    v = np.where(e == 0, f / 8 * 2.0 ** -6, (1 + f / 8) * 2.0 ** (e - 7.0)) * np.where(q > 127, -1, 1)
    v *= np.repeat(np.repeat(s, 128, 0), 128, 1)
    # 131072 values of a law whose fourth moment is below 12 times its variance's square, times scales of 0.8..1.2 (mean
    # square 1.0133): the mean square is within 0.013 + 4 * sqrt(12 / 131072) of 1 / 512, and the eight scales' own spread
    # (0.23 of the square's mean, over 8, four times) 0.33
    assert abs((v * v).mean() * 512 - 1) < 0.013 + 0.04 + 0.33


def test_a_prompt_reaches_the_engine_as_it_is():
    class Engine:
        def start(self, token):
            self.got = token
            return 7, {}
    e = Engine()
    MtpLoop(e).start([1, 2, 3])
    assert e.got == [1, 2, 3]
