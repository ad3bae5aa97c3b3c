"""The F8 experts' h = silu(g) u: quantised from exact block products for every number of rows, and y of them."""
from __future__ import annotations

import numpy as np
import pytest

import f8_ref as ref

pytestmark = pytest.mark.gpu

H, F = 512, 300


@pytest.fixture(scope="module")
def be():
    from turboqwenfare_amd.backend import HipBackend

    with HipBackend(0) as b:
        yield b


def tile_rows(n, t, k, width):
    """Rows of a tile as the library chooses them on 256 compute units; 0: slots by themselves."""
    pairs, blocks = t * k, -(-width // 128)
    if t <= 16 and pairs <= 64:
        return 0
    mean = min(pairs // n, 14) if pairs <= 64 else pairs // n
    if mean <= 14:
        return 16 if mean <= 6 else 32
    if n * -(-mean // 64) * blocks < 128:
        return 32
    if mean <= 40:
        return 64
    return 64 if mean > 96 and pairs // 96 * blocks < 512 else 96


class Cancelling:
    """n experts whose gate and up rows have in each block two products of 448 x 448 that cancel, and beside them six
    small ones; row r of down takes h's column r % F."""

    def __init__(self, be, n):
        rng = np.random.default_rng(n)
        code = np.zeros(1024, np.uint8)  # by value + 448
        for v in (-448, -2, -1, 0, 1, 2, 448):
            code[v + 448] = np.flatnonzero(ref.TABLE == v)[0]
        down = np.zeros((H, F), int)
        down[np.arange(H), np.arange(H) % F] = 1
        self.be, self.small, self.handles = be, [], [[], [], []]
        for _ in range(n):
            pair = []
            for i in range(2):
                m = np.zeros((F, H), int)
                for b in range(0, H, 128):
                    m[:, b + 2:b + 8] = rng.integers(-2, 3, (F, 6))
                pair.append(m.astype(np.float64))
                m[:, 0::128], m[:, 1::128] = 448, -448
                self.handles[i].append(be.upload_f8(code[m + 448], np.full((3, 4), 0.25, np.float32)))
            self.small.append(pair)
            self.handles[2].append(be.upload_f8(code[down + 448], np.ones((4, 3), np.float32)))
        self.ex = be.prepare_f8_experts(*self.handles)

    def close(self):
        self.be.free_f8_experts(self.ex)
        for g in self.handles:
            for w in g:
                self.be.free_weights(w)


@pytest.fixture(scope="module")
def layers(be):
    """Cancelling layers by their number of experts, made when they are asked for."""
    made = {}

    def layer(n):
        if n not in made:
            made[n] = Cancelling(be, n)
        return made[n]

    yield layer
    for one in made.values():
        one.close()


@pytest.mark.parametrize("kind,y_kind", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("n,t,k,m", [
    (2, 1, 1, 0), (2, 5, 1, 0), (2, 12, 2, 0), (2, 17, 1, 32), (2, 40, 1, 32), (2, 100, 1, 32), (2, 400, 1, 32), (2, 4096, 1, 64),
    (24, 16, 1, 0), (24, 100, 1, 16), (24, 300, 1, 32), (24, 2500, 1, 64), (24, 4096, 5, 96),
    (64, 1, 1, 0), (64, 100, 1, 16), (64, 700, 1, 32), (64, 1100, 1, 64), (64, 2500, 1, 64), (64, 3500, 1, 96), (64, 4096, 1, 96)])
def test_h_comes_from_exact_products(be, layers, n, t, k, m, kind, y_kind):
    """Slots by themselves and tiles of every number of rows: h is lost where products are cut."""
    made = layers(n)
    assert tile_rows(n, t, k, F) == m
    rng = np.random.default_rng(t)
    x = np.zeros((t, H), np.float32)
    x[:, 0::128] = x[:, 1::128] = 448
    for b in range(0, H, 128):
        x[:, b + 2:b + 8] = rng.integers(1, 4, (t, 6))
    ids = np.repeat(rng.integers(0, n, (t, 1)), k, 1).astype(np.uint16)  # one expert in all slots of a row
    w = (rng.uniform(0.5, 1, (t, k)) / k).astype(np.float32)
    d = [be.to_device(a) for a in (ref.to_bf16(x) if kind == "bf16" else x, ids, w, np.zeros((t, H), np.uint16 if y_kind == "bf16" else np.float32))]
    be.f8_experts_device(made.ex, d[0], t, d[1], d[2], k, d[3], x_type=kind, y_type=y_kind)
    got = be.read(d[3], np.uint16 if y_kind == "bf16" else np.float32, (t, H))
    got = (ref.from_bf16(got) if y_kind == "bf16" else got).astype(np.float64)
    for b in d:
        be.free(b)
    small_x, total = np.where(x == 448, 0, x).astype(np.float64), w.astype(np.float64).sum(1, keepdims=True)
    for e in range(n):
        rows = ids[:, 0] == e
        if not rows.any():
            continue
        g, u = (0.25 * small_x[rows] @ m.T for m in made.small[e])  # multiples of 1/4, exact in f32
        h = g / (1 + np.exp(-g)) * u
        q, s, _ = ref.quantize(h)
        want = (total[rows] * h)[:, np.arange(H) % F]
        # e4m3 is off by at most half a step (2^-4 of the value, 2^-10 of the scale below 2^-6 of it); h, the scale and
        # the sum by 2^-18; a bf16 y by 2^-8 and a term that waits as f16 by 2^-11 of it and 2^-24 of the block's
        # largest value, of which 448 s is more than half
        step = (2.0 ** -4 * np.abs(h) + 2.0 ** -10 * s)[:, np.arange(H) % F] * total[rows]
        tol = step + 2.0 ** -18 * np.abs(want) + (2.0 ** -8 + 2.0 ** -11) * (np.abs(want) + step)
        tol = tol + 2.0 ** -24 * np.abs(want).max(1, keepdims=True, initial=0)
        assert np.all(np.abs(got[rows] - want) <= tol)


@pytest.mark.parametrize("kind,y_kind", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("n,t,k,m", [(13, 100, 6, 32), (13, 400, 8, 64), (5, 200, 5, 32), (1, 90, 1, 32), (2, 300, 1, 32), (60, 320, 4, 64), (60, 800, 4, 96),
                                     (60, 3200, 4, 64), (60, 4096, 5, 96)])
def test_y_is_as_near_as_its_type(be, n, t, k, m, kind, y_kind):
    """An f32 y element by element within what exact block products allow, and every y on the whole as near as f32 sums
    and its own rounding bring it."""
    from test_gpu_f8 import Layer, rows_of, values_of

    layer = Layer(be, n, 200, 300, n)
    assert tile_rows(n, t, k, 300) == m
    rng = np.random.default_rng(t)
    bits = rows_of(rng, t, 200, kind)
    ids, w = layer.routes(rng, t, k)
    got, st = layer.run(bits, kind, ids, w, y_kind)
    assert st == 0
    got = values_of(got, y_kind).astype(np.float64)
    want, tol = ref.experts(values_of(bits, kind), ids, w, layer.mats, False, y_kind)
    if y_kind == "f32":
        assert np.all(np.abs(got - want) <= tol + 1e-35)
    # With e the 2-norm error of g and u, that of y is sqrt(e / 4): a value of h is off by about 2 e z before its rounding
    # and passes the middle of two steps (z / 8 at most) with a chance of that over the step.  f32 sums of up to 300
    # products add up to sqrt(300) roundings of 2^-24, so e <= 1.1e-6 and y is off by at most 5.2e-4.  A bf16 y is off by
    # its rounding, even on +-2^-8 of a value's power of two, so 2^-8 / sqrt(3) of the values at most; its terms by that of
    # f16, 2^-11 / sqrt(3) of theirs, whose norm is at most twice that of the sum here; and by 3.9e-5 of the fp8 cores.
    whole = 5.2e-4 if y_kind == "f32" else (5.2e-4 ** 2 + (2.0 ** -16 + 2.0 ** -20) / 3) ** 0.5 + 3.9e-5
    assert np.linalg.norm(got - want) <= whole * np.linalg.norm(want), np.linalg.norm(got - want) / np.linalg.norm(want)
    layer.close()


def test_large_tiles(be):
    """Tiles of 64 and 96 rows: uneven routes, empty slots, off alignment, rows that are no numbers, other orders, an expert
    that is not there."""
    from test_gpu_f8 import Layer

    n, hidden, width = 60, 331, 290
    layer = Layer(be, n, hidden, width, 9)
    for t, k, m in ((300, 4, 64), (800, 5, 96), (3000, 4, 64), (4096, 5, 96)):
        assert tile_rows(n, t, k, width) == m
        layer.check(t, k, "bf16", "bf16", skew=1.2, empty=0.2, offset=1)
        layer.check(t, k, "f32", "f32", skew=0.4, offset=3)
    for t, k, y_kind in ((300, 4, "bf16"), (300, 4, "f32"), (900, 5, "bf16"), (900, 5, "f32")):
        rng = np.random.default_rng(t)
        x = rng.standard_normal((t, hidden)).astype(np.float32)
        ids, w = layer.routes(rng, t, k, empty=0.0)
        clean, _ = layer.run(x, "f32", ids, w, y_kind)
        x[1, 5], x[t - 1, 0] = np.nan, np.inf
        got, st = layer.run(x, "f32", ids, w, y_kind)
        rest = ~np.isin(np.arange(t), [1, t - 1])
        value = ref.from_bf16(got) if y_kind == "bf16" else got
        assert st == 0 and np.isnan(value[~rest]).all() and np.array_equal(got[rest], clean[rest])
        p = rng.permutation(t)
        shuffled, _ = layer.run(np.ascontiguousarray(x[p]), "f32", np.ascontiguousarray(ids[p]), np.ascontiguousarray(w[p]), y_kind)
        assert np.array_equal(shuffled[np.isin(p, np.flatnonzero(rest))], got[p][np.isin(p, np.flatnonzero(rest))])
        ids[t // 2, k - 1] = n
        y, st = layer.run(x, "f32", ids, w, y_kind)
        assert st == 1 and (y == (0x4242 if y_kind == "bf16" else 7)).all()
    layer.close()


@pytest.mark.parametrize("hidden,width", [(65536, 5), (5, 65536)])
def test_as_wide_as_any(be, hidden, width):
    """512 blocks of K, by few slots and by tiles."""
    from test_gpu_f8 import Layer

    layer = Layer(be, 2, hidden, width, 3)
    for t, k in ((1, 2), (17, 2), (130, 1)):
        layer.check(t, k, "bf16", "f32")
        layer.check(t, k, "f32", "bf16")
    layer.close()


def test_as_many_experts_as_any(be):
    """1024 experts (that take turns with 16 matrices each), one slot to an expert and 64."""
    from test_gpu_f8 import Layer

    few = Layer(be, 16, 130, 70, 4)
    n = 1024
    many = Layer.__new__(Layer)
    many.be, many.n, many.hidden, many.width = be, n, few.hidden, few.width
    many.mats = [few.mats[e % 16] for e in range(n)]
    many.ex = be.prepare_f8_experts(*([g[e % 16] for e in range(n)] for g in few.handles))
    for t, k in ((1, 16), (64, 16), (4096, 5), (4096, 16)):
        many.check(t, k, "bf16", "bf16")
    be.free_f8_experts(many.ex)
    few.close()
