"""Heads before the attention on the GPU: norms, rotation and the cache against their definitions in 64 bits
(attn_ref.py), and what the calls refuse."""
from __future__ import annotations

import numpy as np
import pytest

import attn_ref as ref
import f8_ref
from turboqwenfare_amd._lib import ERR_INVALID, HipError

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    from turboqwenfare_amd.backend import HipBackend

    with HipBackend(0) as b:
        yield b


def given(x, kind):
    """(what the call gets, its values in 64 bits)"""
    x = np.ascontiguousarray(x, np.float32)
    if kind == "f32":
        return x, x.astype(np.float64)
    bits = f8_ref.to_bf16(x)
    return bits, f8_ref.from_bf16(bits).astype(np.float64)


def near(got, want, tol):
    bad = ~(np.abs(got - want) <= tol) & ~(np.isnan(got) & np.isnan(want))
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4], tol[bad][:4])


FREQ = lambda n: 1e6 ** (-np.arange(n) / max(n, 1))  # noqa: E731


class Case:
    """A call over rows of one projection [t, q_heads + 2 kv_heads (+ a gap), d], with guards behind every output."""

    def __init__(self, be, t, heads, kind, pairs=0, order="half", norms=True, cache=None, page=16, seed=0, gap=0, first=0, eps=1e-6, x=None):
        self.be, self.t, self.heads, self.order = be, t, heads, order
        nq, nk, d = heads
        rng = np.random.default_rng(seed)
        x = rng.standard_normal((t, nq + 2 * nk, d + gap)) * np.exp2(rng.integers(-6, 6, (t, 1, 1))) if x is None else x
        bits, values = given(x, kind)
        size, row = bits.itemsize, (nq + 2 * nk) * (d + gap)
        self.q64, self.k64, self.v64 = values[:, :nq, :d], values[:, nq:nq + nk, :d], values[:, nq + nk:, :d]
        self.wq, self.wk = [(1 + 0.2 * rng.standard_normal(d)).astype(np.float32) if norms else None for _ in range(2)]
        self.pos = (first + rng.permutation(2 * t)[:t]).astype(np.int32)
        self.freq, self.eps = FREQ(pairs), eps
        self.keep = []
        dev = self.dev
        whole = dev(bits)
        at = lambda h: be.view(whole, h * (d + gap) * size, whole.nbytes - h * (d + gap) * size)  # noqa: E731
        self.n_pages = -(-t // page) + 2
        rng2 = np.random.default_rng(seed + 1)
        self.slots = rng2.permutation(self.n_pages * page)[:t].astype(np.int32)
        self.q_out, self.k_out, self.v_out = [dev(np.full(t * n * d + 8, 0x7FFF, np.uint16)) for n in (nq, nk, nk)]
        self.cache = None
        if cache:
            n = self.n_pages * nk * page
            bytes_ = np.full(n * d * (1 if cache == "f8" else 2), 0x55, np.uint8)
            self.cache = be.kv_cache(dev(bytes_), dev(bytes_), self.n_pages, nk, page, d, cache,
                                     *([dev(np.full(n, 9.0, np.float32)) for _ in range(2)] if cache == "f8" else []))
        self.status = dev(np.zeros(1, np.int32))
        self.rope = be.prepare_rope(self.freq) if pairs else None
        self.norms = [be.upload_f32(w) if w is not None else None for w in (self.wq, self.wk)]
        self.args = dict(d_q=at(0), d_k=at(nq), d_v=at(nq + nk), t=t, heads=heads, d_positions=dev(self.pos), d_q_out=self.q_out,
                         d_k_out=self.k_out, d_v_out=self.v_out, x_type=kind, strides=((row, d + gap),) * 3, q_norm=self.norms[0],
                         k_norm=self.norms[1], eps=eps, rope=self.rope, pairs=order, cache=self.cache,
                         d_slots=dev(self.slots) if cache else None, d_status=self.status)

    def dev(self, a):
        self.keep.append(self.be.to_device(a))
        return self.keep[-1]

    def run(self, **changed):
        self.be.qk_rope_device(**{**self.args, **changed})

    def read(self, buf, n):
        a = self.be.read(buf, np.uint16, (self.t * n * self.heads[2] + 8,))
        assert (a[-8:] == 0x7FFF).all()
        return f8_ref.from_bf16(a[:-8]).astype(np.float64).reshape(self.t, n, self.heads[2])

    def wanted(self):
        q, tq = ref.heads_after(self.q64, self.wq, self.eps, self.pos, self.freq, self.order)
        k, tk = ref.heads_after(self.k64, self.wk, self.eps, self.pos, self.freq, self.order)
        return (q, tq), (k, tk), (self.v64, np.zeros_like(self.v64))

    def check(self):
        for got, (want, tol) in zip((self.read(b, n) for b, n in zip((self.q_out, self.k_out, self.v_out), (self.heads[0], self.heads[1], self.heads[1]))),
                                    self.wanted()):
            near(got, want, tol + (np.abs(want) + tol) * ref.BF16)

    def cached(self, which):
        """(values f64 [t, heads, d] at the rows' slots, scales, raw bytes elsewhere are untouched)"""
        c, be = self.cache, self.be
        nk, d, page = self.heads[1], self.heads[2], c.page_size
        buf = c.d_k if which == "k" else c.d_v
        f8 = c.type == "f8"
        raw = be.read(buf, np.uint8 if f8 else np.uint16, (self.n_pages, nk, page, d)).transpose(0, 2, 1, 3).reshape(-1, nk, d)
        used = np.zeros(len(raw), bool)
        used[self.slots[self.slots >= 0]] = True
        assert (raw[~used] == (0x55 if f8 else 0x5555)).all()
        if not f8:
            return f8_ref.from_bf16(np.ascontiguousarray(raw[self.slots])).astype(np.float64), None
        s = be.read(c.d_k_scales if which == "k" else c.d_v_scales, np.float32, (self.n_pages, nk, page)).transpose(0, 2, 1).reshape(-1, nk)
        assert (s[~used] == 9.0).all()
        return f8_ref.TABLE[raw[self.slots]] * s[self.slots].astype(np.float64)[..., None], s[self.slots].astype(np.float64)

    def check_cache(self):
        _, k, v = self.wanted()
        for which, (want, tol) in (("k", k), ("v", v)):
            got, scale = self.cached(which)
            if scale is None:
                near(got, want, tol + (np.abs(want) + tol) * ref.BF16)
            else:
                # half a step of e4m3 (2^-4 of the value, 2^-10 of the scale below 2^-6 of it), of what f32 gave
                near(scale, np.abs(want).max(2) / 448, tol.max(2) / 448 + np.abs(want).max(2) / 448 * 2.0 ** -22)
                near(got, want, tol + np.maximum((np.abs(want) + tol) * 2.0 ** -4, scale[..., None] * 2.0 ** -10) * (1 + 2.0 ** -20))

    def free(self):
        for b in self.keep:
            self.be.free(b)
        if self.rope:
            self.be.free_rope(self.rope)
        for w in self.norms:
            if w:
                self.be.free_tensor(w)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("order", ["half", "neighbours"])
@pytest.mark.parametrize("heads,pairs,t", [
    ((16, 2, 256), 32, 1), ((16, 2, 256), 32, 37), ((32, 8, 128), 64, 5), ((8, 8, 64), 32, 9), ((1, 1, 64), 8, 3), ((6, 3, 128), 24, 17),
    ((5, 1, 256), 128, 2), ((7, 7, 256), 8, 4), ((4, 2, 64), 16, 515)])
def test_heads(be, kind, order, heads, pairs, t):
    c = Case(be, t, heads, kind, pairs, order, cache="bf16", seed=t, gap=8 if t % 2 else 0)
    c.run()
    c.check()
    c.check_cache()
    assert be.read(c.status, np.int32, (1,))[0] == 0
    c.free()


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("heads", [(16, 2, 256), (4, 4, 128), (2, 1, 64)])
def test_e4m3_cache(be, page, heads):
    c = Case(be, 50, heads, "f32", 16, "half", cache="f8", page=page, seed=page)
    c.run()
    c.check()
    c.check_cache()
    c.free()


def test_without_norms_rotation_or_cache(be):
    """q and v are then their inputs, rounded."""
    c = Case(be, 11, (3, 1, 128), "f32", 0, "half", norms=False, seed=3)
    c.run(d_positions=None)
    c.check()
    c.run(d_k_out=None, d_v_out=None, d_positions=None)
    c.free()


def test_far_positions(be):
    """Angles of positions near 2^30, whose f32 would be whole turns off; and negative ones."""
    for first in (2 ** 30, -2 ** 20):
        c = Case(be, 9, (2, 1, 128), "f32", 64, "half", seed=5, first=first)
        c.run()
        # the angle's 64-bit product itself: 2^30 * 2^-53 turns
        c.check()
        c.free()


def test_zero_rows_and_odd_values(be):
    """A zero head stays zero (also with e4m3, whose scale is 0); a NaN or an infinity stays in its head."""
    x = np.random.default_rng(0).standard_normal((4, 6, 64)).astype(np.float32)
    x[0] = 0.0
    x[1, 1, 3], x[2, 4, 5], x[3, 5, 7] = np.nan, np.inf, np.nan
    for cache in ("bf16", "f8"):
        c = Case(be, 4, (2, 2, 64), "f32", 32, "half", cache=cache, x=x)
        c.run()
        q, k, v = c.read(c.q_out, 2), c.read(c.k_out, 2), c.read(c.v_out, 2)
        assert (q[0] == 0).all() and (k[0] == 0).all() and (v[0] == 0).all()
        assert np.isnan(q[1, 1]).all() and np.isfinite(q[1, 0]).all() and np.isfinite(q[[0, 2, 3]]).all()
        assert np.isfinite(k).all() and np.isinf(v[2, 0, 5]) and np.isnan(v[3, 1, 7])
        kc, vc = c.cached("k")[0], c.cached("v")[0]
        assert (kc[0] == 0).all() and (vc[0] == 0).all() and np.isfinite(kc).all() and np.isfinite(vc[:2]).all()
        if cache == "f8":
            assert np.isnan(vc[2, 0, 5]) and np.isnan(vc[3, 1, 7]) and np.isfinite(vc[2, 1]).all() and np.isfinite(vc[3, 0]).all()
        else:
            assert np.isinf(vc[2, 0, 5]) and np.isnan(vc[3, 1, 7])
        c.free()


def test_rows_without_a_slot(be):
    """Slot -1 is not cached; one outside the cache neither, and it is reported."""
    c = Case(be, 6, (2, 2, 64), "bf16", 16, "half", cache="bf16")
    c.slots[[1, 4]] = -1
    be.write(c.args["d_slots"], c.slots)
    c.run()
    assert be.read(c.status, np.int32, (1,))[0] == 0
    _, (k, tol), _ = c.wanted()
    got = c.cached("k")[0]
    real = c.slots >= 0
    near(got[real], k[real], (tol + (np.abs(k) + tol) * ref.BF16)[real])
    c.check()
    for wrong in (c.n_pages * 16, -2, 2 ** 31 - 1):
        be.write(c.status, np.zeros(1, np.int32))
        c.slots[4] = wrong
        be.write(c.args["d_slots"], c.slots)
        c.run()
        assert be.read(c.status, np.int32, (1,))[0] == ERR_INVALID
        c.slots[4] = -1
        c.cached("k")
    c.free()


def test_cache_past_32_bits(be):
    """Slots whose elements lie behind 2^32 bytes."""
    page, nk, d = 256, 8, 256
    n_pages = 2 ** 32 // (page * nk * d * 2) + 3
    c = Case(be, 3, (8, nk, d), "bf16", 32, "half", seed=8)
    k, v = be.alloc(n_pages * page * nk * d * 2), be.alloc(n_pages * page * nk * d * 2)
    cache = be.kv_cache(k, v, n_pages, nk, page, d)
    slots = np.array([n_pages * page - 1, 5, (n_pages - 2) * page + 17], np.int32)
    c.run(cache=cache, d_slots=c.dev(slots))
    _, (kw, tol), _ = c.wanted()
    for row, s in enumerate(slots):
        for h in range(nk):
            at = (((int(s) // page) * nk + h) * page + int(s) % page) * d * 2
            got = f8_ref.from_bf16(be.read(be.view(k, at, d * 2), np.uint16, (d,))).astype(np.float64)
            near(got, kw[row, h], tol[row, h] + (np.abs(kw[row, h]) + tol[row, h]) * ref.BF16)
    for b in (k, v):
        be.free(b)
    c.free()


def test_refusals(be):
    c = Case(be, 4, (4, 2, 64), "f32", 32, "half", cache="f8")
    a = c.args

    def refused(**changed):
        with pytest.raises((HipError, ValueError)) as e:
            c.run(**changed)
        assert not isinstance(e.value, HipError) or e.value.status == ERR_INVALID

    for heads in ((0, 0, 64), (4, 3, 64), (4, 2, 96), (4, 0, 64)):
        refused(heads=heads)
    for t in (0, 65537):
        refused(t=t)
    refused(eps=-1.0)
    refused(eps=float("nan"))
    refused(x_type="f16")
    refused(pairs="other")
    refused(strides=((12, 64), None, None))       # rows that are not aligned
    refused(strides=((512, 4), None, None))
    refused(strides=((32, 64), None, None))       # rows inside one another
    refused(strides=((2 ** 24, 64), None, None))
    refused(d_q=be.view(a["d_q"], 4, a["d_q"].nbytes - 4))
    refused(d_positions=None)
    refused(cache=None)
    refused(d_slots=None)
    refused(d_q_out=a["d_q"])                     # in place
    refused(d_k_out=a["d_v_out"])
    refused(d_v_out=c.cache.d_v)
    refused(d_q_out=be.view(c.q_out, 2, c.q_out.nbytes - 2))
    wrong = be.upload_f32(np.ones(65, np.float32))
    refused(q_norm=wrong)
    wide = be.prepare_rope(np.ones(40))
    refused(rope=wide)
    for bad in ([], np.ones(4), np.ones(136), [np.inf] * 8):
        with pytest.raises(HipError):
            be.prepare_rope(bad)
    import dataclasses
    for changed in (dict(page_size=8), dict(page_size=48), dict(page_size=512), dict(kv_heads=1), dict(head_dim=128), dict(n_pages=0),
                    dict(n_pages=2 ** 27), dict(d_k_scales=None), dict(d_k=be.view(c.cache.d_k, 8, 8))):
        refused(cache=dataclasses.replace(c.cache, **changed))
    with pytest.raises(ValueError):
        be.kv_cache(c.cache.d_k, c.cache.d_v, 1000, 2, 16, 64)
    be.free_tensor(wrong)
    be.free_rope(wide)
    assert (be.read(c.q_out, np.uint16, (8,)) == 0x7FFF).all()
    c.run()
    c.check()
    c.free()


def test_add_rows(be):
    rng = np.random.default_rng(1)
    for n in (1, 255, 256, 1000, 70001):
        a, b = rng.standard_normal((2, n)).astype(np.float32)
        da, db, do = be.to_device(a), be.to_device(b), be.to_device(np.full(n + 1, 5.0, np.float32))
        be.add_rows_device(da, db, n, do)
        got = be.read(do, np.float32, (n + 1,))
        assert np.array_equal(got[:n], a + b) and got[n] == 5.0
        be.add_rows_device(da, db, n, da)  # in place
        assert np.array_equal(be.read(da, np.float32, (n,)), a + b)
        be.add_rows_device(db, db, n, db)
        assert np.array_equal(be.read(db, np.float32, (n,)), b + b)
        with pytest.raises(HipError):
            be.add_rows_device(da, db, 0, do)
        if n > 2:
            with pytest.raises(HipError):
                be.add_rows_device(da, db, n - 1, be.view(da, 4, 4 * (n - 1)))
        for x in (da, db, do):
            be.free(x)
