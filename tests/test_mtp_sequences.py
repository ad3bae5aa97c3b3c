"""Whose sequence a model's attention caches hold: after prompts that are refused, and after passes that fail (on the CPU)."""
from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest

from test_attention_layers import SMALL, Recorder
from turboqwenfare_amd import attention
from turboqwenfare_amd.attention import AttentionLayers
from turboqwenfare_amd.mtp_loop import DeviceEngine

VOCAB, K = 50, 3


class Device(Recorder):
    """Reads give zeros, and `status` where a status is read; the call named `broken` raises."""

    status, broken = 0, None

    def write(self, buf, a):
        self.calls.append(("write", (buf, a), {}))

    def read(self, buf, kind, shape):
        return np.full(shape, self.status if buf.nbytes == 4 and kind == np.int32 else 0, kind)

    def __getattr__(self, name):
        call = super().__getattr__(name)
        if name == self.broken:
            raise RuntimeError(name)
        return call


def engines(n, **changed):
    be = Device()
    layers = AttentionLayers(be, 1, **{**SMALL, **changed})
    model = SimpleNamespace(vocab=VOCAB, n_layers=1, attention=layers, parts=[SimpleNamespace(stack=None)], draft=SimpleNamespace(stack=None), embed=None,
                            norm=None, draft_norm=None, lm_head=None)
    return be, layers, [DeviceEngine(be, model, k=K, greedy=True) for _ in range(n)]


def positions(be):
    """(first, rows) of the attention's passes since the last look."""
    got = [(c[1][5].ptr, c[1][3]) for c in be.calls if c[0] == "qk_rope_device"]
    be.calls.clear()
    return got


@pytest.mark.parametrize("bad", [[], [VOCAB], [3, -1], [1] * (SMALL["max_tokens"] + 1)], ids=["empty", "unknown", "negative", "too_long"])
def test_a_refused_prompt_changes_nothing(bad):
    be, layers, (a, b) = engines(2)
    a.start([1] * 9)
    for other in (a, b):
        with pytest.raises(ValueError):
            other.start(bad)
    be.calls.clear()
    a.plain(0, 1)
    a.speculative(1, 1)
    at = layers.d_count.ptr
    assert positions(be) == [(at + 4 * 9, 1), (at + 4 * 10, K + 1)] and a.length == 11 and layers.sequence is a
    for call in (b.plain, b.speculative):  # nothing of it is in the caches
        with pytest.raises(RuntimeError):
            call(0, 1)
    assert positions(be) == []


def test_prompts_longer_than_the_projections_take(monkeypatch):
    monkeypatch.setattr(attention, "F8_MAX_TOKENS", 20)
    be, layers, (a, b) = engines(2)
    a.start([1] * 20)
    be.calls.clear()
    with pytest.raises(ValueError):
        b.start([1] * 21)
    with pytest.raises(ValueError):
        layers.forward(0, b.d_h, 21, 0)
    assert be.calls == [] and layers.sequence is a
    a.plain(0, 1)


@pytest.mark.parametrize("what", ["status", "f8_matmul_device", "lm_head_logits_device"])
def test_a_prompt_pass_that_fails_leaves_no_sequence(what):
    """The caches hold a part of the new prompt: neither engine goes on."""
    be, layers, (a, b) = engines(2)
    a.start([1] * 9)
    if what == "status":
        be.status = -1
    else:
        be.broken = what
    with pytest.raises(RuntimeError):
        b.start([1] * 12)
    be.status, be.broken = 0, None
    be.calls.clear()
    for call in (a.plain, a.speculative, b.plain, b.speculative):
        with pytest.raises(RuntimeError, match="sequence"):
            call(0, 1)
    assert positions(be) == [] and layers.sequence is None
    a.start([1] * 9)
    a.plain(0, 1)


@pytest.mark.parametrize("step", ["plain", "speculative"])
def test_a_step_that_fails_can_be_made_again(step):
    """What it wrote stands behind the sequence."""
    be, layers, (a,) = engines(1)
    a.start([1] * 9)
    be.broken = "lm_head_logits_device"
    with pytest.raises(RuntimeError):
        getattr(a, step)(0, 1)
    be.broken = None
    be.calls.clear()
    getattr(a, step)(0, 1)
    assert positions(be)[0] == (layers.d_count.ptr + 4 * 9, 1 if step == "plain" else K + 1)
