"""The expert handles of perf/operators.py live as long as the states that use them (on the CPU, with a library that
counts)."""
from __future__ import annotations

import gc
import importlib.util
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent


class Counting:
    """Handles are numbers; those given back are remembered, and the order."""

    def __init__(self):
        self.made, self.freed, self.experts, self.ran = 0, [], {}, []

    def _new(self):
        self.made += 1
        return self.made

    def upload_f8_device(self, q, s, rows, cols):
        return self._new()

    def prepare_f8_experts(self, gate, up, down):
        h = self._new()
        self.experts[h] = [*gate, *up, *down]
        return h

    def free_f8_experts(self, h):
        assert h in self.experts and h not in self.freed and not set(self.experts[h]) & set(self.freed)
        self.freed.append(h)

    def free_weights(self, h):
        assert h not in self.freed
        self.freed.append(h)

    def f8_experts_device(self, h, *args, **kwargs):
        assert h in self.experts and h not in self.freed and not set(self.experts[h]) & set(self.freed)
        self.ran.append(h)


@pytest.fixture
def operators(monkeypatch):
    spec = importlib.util.spec_from_file_location("operators_under_test", ROOT / "perf" / "operators.py")
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.DEV, m.own = "cpu", True
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    library = Counting()
    monkeypatch.setattr(m, "_backend", lambda: library)
    yield m, library


def case(experts, hidden, layers=1):
    return dict(kind="experts", t=3, hidden=hidden, width=64, experts=experts, top_k=2, skew=0.0, empty=0.0, layers=layers, x="f32")


def test_a_state_keeps_its_handles(operators):
    m, library = operators
    a = m.prepare(case(4, 128, 2), 0)
    made = library.made
    again = m.prepare(case(4, 128, 2), 1)  # the same weights, laid out once
    assert library.made == made
    b = m.prepare(case(3, 256), 0)
    for state in (a, b, again, a):  # another geometry in between
        m.run(state)
    first = set(library.experts[library.ran[0]]) | {library.ran[0]}
    assert not library.freed
    del a
    gc.collect()
    m.run(again)
    assert not library.freed
    del again, state
    gc.collect()
    assert first <= set(library.freed) and len(library.freed) == made
    m.run(b)


def test_the_newest_geometry_is_kept(operators):
    m, library = operators
    for seed in range(3):
        m.run(m.prepare(case(4, 128), seed))
        gc.collect()
    assert library.made == 13 and not library.freed
