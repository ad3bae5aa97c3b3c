"""perf/more_operators.py on the CPU: the plain forms against the definitions, what is drawn, and that handles live as
long as the states that use them."""
from __future__ import annotations

import gc
import importlib.util
import random
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture
def more(monkeypatch):
    spec = importlib.util.spec_from_file_location("more_operators_under_test", ROOT / "perf" / "more_operators.py")
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.DEV = "cpu"
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    return m


HEADS = dict(q_heads=4, kv_heads=2, dim=64)
CASES = [
    dict(kind="rope", t=5, **HEADS, rotary=32, pairs="half", x="f32", packed=True, page=16),
    dict(kind="rope", t=18, **HEADS, rotary=64, pairs="neighbours", x="bf16", packed=False, page=16),
    dict(kind="rope", t=3, **HEADS, rotary=0, pairs="half", x="f32", packed=True, page=16),
    dict(kind="prompt", seqs=1, low=7, high=7, context=0, **HEADS, gate=True),
    dict(kind="prompt", seqs=5, low=1, high=30, context=9, **HEADS, gate=False),
    dict(kind="paged", seqs=3, rows=2, low=8, high=60, **HEADS, page=16, cache="bf16", gate=True),
    dict(kind="paged", seqs=2, rows=1, low=8, high=40, **HEADS, page=16, cache="f8", gate=False),
]


def pairs_of(a, b):
    if isinstance(a, dict):
        for k in a:
            if a[k] is not None:
                yield a[k], b[k]
    else:
        yield a, b


@pytest.mark.parametrize("case", CASES, ids=lambda c: c["kind"])
def test_plain_forms_are_the_definitions(more, case):
    """Outputs are rounded to bf16 once: half a step, 2^-8 of the value; the arithmetic before it is 32-bit (the 2^-16 of
    the largest value is far above its sums of 64 and of 60 terms)."""
    out, want = more.run(more.prepare(case, 3)), more.exact(case, 3)
    for got, exact in pairs_of(out, want):
        got = got.double()
        assert got.shape == exact.shape and torch.isfinite(got).all() and got.abs().max() > 0
        assert ((got - exact).abs() <= exact.abs() * 2.0 ** -8 + exact.abs().max() * 2.0 ** -16).all()


def test_inputs_follow_the_seed(more):
    for case in CASES:
        a, b, c = more.prepare(case, 1), more.prepare(case, 1), more.prepare(case, 2)
        assert torch.equal(a["q"], b["q"]) and not torch.equal(a["q"], c["q"])


def test_listed_cases(more):
    cases = more.listed()
    names = [c["name"] for c in cases]
    assert len(set(names)) == len(names) and {c["kind"] for c in cases} == {"rope", "prompt", "paged"}
    for c in cases:
        w = more.work(c)
        assert w["bytes"] > 0 and w["flops"] > 0


def test_draws_are_cases_the_calls_take(more):
    rng = random.Random(5)
    largest = {k: max(more.work(c)["bytes"] + more.work(c)["flops"] / 240 for c in more.listed() if c["kind"] == k) for k in ("rope", "prompt", "paged")}
    seen = set()
    for _ in range(300):
        c = more.draw(rng)
        assert c["q_heads"] % c["kv_heads"] == 0 and 1 <= c["q_heads"] <= 256 and c["dim"] in (64, 128, 256)
        seen.add((c["kind"], c["dim"]))
        if c["kind"] == "rope":
            assert 1 <= c["t"] <= 4096 and c["rotary"] % 16 == 0 and c["rotary"] <= c["dim"]
            continue
        lens = more._lengths(c)
        assert len(lens) == c["seqs"] and max(lens) == c["high"] and min(lens) >= min(c["low"], c["high"])
        if c["kind"] == "paged":
            assert c["rows"] <= 8 <= min(lens)
        w = more.work(c)
        assert w["bytes"] + w["flops"] / 240 < 4 * largest[c["kind"]]
    assert len(seen) == 9


class Counting:
    """Handles are numbers; those given back are remembered."""

    def __init__(self):
        self.made, self.freed = 0, []

    def _new(self, *args, **kwargs):
        self.made += 1
        return self.made

    upload_f32 = prepare_rope = _new

    def kv_cache(self, *args, **kwargs):
        return object()

    def _free(self, h):
        assert h not in self.freed
        self.freed.append(h)

    free_tensor = free_rope = _free

    def qk_rope_device(self, *args, q_norm, k_norm, rope, **kwargs):
        assert not {q_norm, k_norm, rope} & set(self.freed)


def test_handles_live_as_long_as_their_state(more, monkeypatch):
    library = Counting()
    monkeypatch.setattr(more, "_backend", lambda: library)
    more.own = True
    states = [more.prepare(CASES[0], s) for s in range(2)]
    for st in states:
        more.run(st)
    del st
    assert library.made == 6 and library.freed == []
    del states[0]
    gc.collect()
    assert len(library.freed) == 3
    more.run(states[0])
    del states
    gc.collect()
    assert sorted(library.freed) == list(range(1, 7))
