"""Attention over the paged cache on the GPU against its definition in 64 bits (attn_ref.py), and what it refuses."""
from __future__ import annotations

import dataclasses

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


def bf16(x):
    bits = f8_ref.to_bf16(np.ascontiguousarray(x, np.float32))
    return bits, f8_ref.from_bf16(bits).astype(np.float64)


class Case:
    def __init__(self, be, lens, rows, heads, kind="bf16", page=16, gate=False, seed=0, gap=0, spare=1, sharp=1.0, change=None):
        self.be, self.heads, self.rows, self.lens = be, heads, rows, list(lens)
        nq, nk, d = heads
        rng = np.random.default_rng(seed)
        need = [-(-n // page) for n in lens]
        n_pages, width = sum(need) + 2, max(max(need), 1) + spare
        order = rng.permutation(n_pages)
        self.table = np.full((len(lens), width), 2 ** 30, np.int32)  # behind a sequence's end: nothing that may be read
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        shape = (n_pages, nk, page, d)
        t = len(lens) * rows
        q, g = rng.standard_normal((t, nq, d + gap)) * sharp, rng.standard_normal((t, nq, d + gap))
        (qb, self.q), (gb, self.gate) = bf16(q), bf16(g)
        self.q, self.gate = self.q[..., :d], self.gate[..., :d] if gate else None
        if kind == "f8":
            kb, ks, self.k = ref.f8_cache(rng, shape)
            vb, vs, self.v = ref.f8_cache(rng, shape)
        else:
            (kb, self.k), (vb, self.v), ks, vs = bf16(rng.standard_normal(shape)), bf16(rng.standard_normal(shape)), None, None
        if change:
            change(self, kb, vb, ks, vs)
            if kind == "f8":
                with np.errstate(invalid="ignore"):
                    self.k, self.v = [f8_ref.TABLE[b] * s[..., None].astype(np.float64) for b, s in ((kb, ks), (vb, vs))]
            else:
                self.k, self.v = [f8_ref.from_bf16(b).astype(np.float64) for b in (kb, vb)]
        self.keep = []
        dev = self.dev
        self.cache = be.kv_cache(dev(kb), dev(vb), n_pages, nk, page, d, kind, *([dev(ks), dev(vs)] if kind == "f8" else []))
        self.y, self.status = dev(np.full(t * nq * d + 8, 0x1234, np.uint16)), dev(np.zeros(1, np.int32))
        st = (nq * (d + gap), d + gap)
        self.args = dict(d_q=dev(qb), heads=heads, n_seqs=len(lens), rows=rows, cache=self.cache, d_pages=dev(self.table), max_pages=width,
                         d_lens=dev(np.array(lens, np.int32)), d_y=self.y, q_strides=st, d_status=self.status,
                         **(dict(d_gate=dev(gb), gate_strides=st) if gate else {}))

    def dev(self, a):
        self.keep.append(self.be.to_device(a))
        return self.keep[-1]

    def token(self, s, j):
        """(page, slot) of token j of sequence s"""
        return self.table[s, j // self.cache_page], j % self.cache_page

    @property
    def cache_page(self):
        return self.page if hasattr(self, "page") else self.cache.page_size

    def run(self, **changed):
        self.be.attn_paged_device(**{**self.args, **changed})
        nq, _, d = self.heads
        t = len(self.lens) * self.rows
        raw = self.be.read(self.y, np.uint16, (t * nq * d + 8,))
        assert (raw[-8:] == 0x1234).all()
        self.raw = raw[:-8].reshape(t, nq, d)
        return f8_ref.from_bf16(self.raw).astype(np.float64)

    def check(self, scale=None):
        s = self.heads[2] ** -0.5 if scale is None else scale
        got = self.run(scale=scale)
        want, tol = ref.paged(self.q, self.k, self.v, self.table, self.lens, self.rows, s, self.gate)
        same = (np.isnan(got) & np.isnan(want)) | (got == want)
        bad = ~(np.abs(got - want) <= tol) & ~same
        assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], tol[bad][:5])
        assert self.be.read(self.status, np.int32, (1,))[0] == 0
        return got

    def free(self):
        for b in self.keep:
            self.be.free(b)


HEADS = [(16, 2, 256), (8, 2, 128), (4, 4, 64), (6, 2, 64), (7, 1, 128), (1, 1, 256), (32, 1, 64), (24, 1, 128)]


@pytest.mark.parametrize("kind", ["bf16", "f8"])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("rows", [1, 4])
def test_one_sequence(be, kind, heads, rows):
    for n in (1, 2, 15, 16, 17, 31, 33, 100, 128, 129, 300, 1100):
        c = Case(be, [n], rows, heads, kind, seed=n, gate=n % 2 == 0)
        c.check()
        c.free()


@pytest.mark.parametrize("kind", ["bf16", "f8"])
@pytest.mark.parametrize("heads,rows", [(h, r) for h, r in zip(HEADS, (2, 8, 3, 5, 8, 7, 8, 2))])
@pytest.mark.parametrize("page", [16, 32, 256])
def test_batch(be, kind, heads, rows, page):
    """Lengths of 0 (no keys), below the rows (first rows without keys), ends inside pages and steps, long beside short."""
    c = Case(be, [0, 1, 3, 700, 16, 5, 129, 0, 2500, 64], rows, heads, kind, page, gate=True, seed=page, gap=8)
    got = c.check()
    assert (got[:rows] == 0).all() and (got[7 * rows:8 * rows] == 0).all() and (got[rows:2 * rows - 1] == 0).all()
    c.free()


@pytest.mark.parametrize("kind", ["bf16", "f8"])
def test_many_sequences(be, kind):
    """More (sequence, key head) than workgroups, more sequences than a wavefront looks through at once."""
    rng = np.random.default_rng(0)
    c = Case(be, rng.integers(0, 90, 700).tolist(), 1, (4, 2, 64), kind, seed=1)
    c.check()
    c.free()


@pytest.mark.parametrize("kind", ["bf16", "f8"])
@pytest.mark.parametrize("heads", [(16, 2, 256), (8, 2, 128), (2, 2, 64)])
def test_long(be, kind, heads):
    """Cut into many parts, beside short ones."""
    c = Case(be, [9000, 40, 20000, 1], 2, heads, kind, 64, seed=2)
    c.check()
    c.free()


@pytest.mark.parametrize("heads", [(2, 1, 256), (2, 1, 128), (2, 1, 64)])
def test_sharp_and_flat_softmax(be, heads):
    for sharp in (0.0, 30.0):
        c = Case(be, [777, 5, 3000], 3, heads, seed=3, sharp=sharp)
        c.check()
        c.check(scale=0.7)
        c.free()


@pytest.mark.parametrize("kind", ["bf16", "f8"])
@pytest.mark.parametrize("heads", [(16, 2, 256), (4, 2, 128), (4, 2, 64)])
def test_odd_values_stay_with_the_rows_that_see_them(be, kind, heads):
    """NaN and infinities behind a sequence's end, in a draft's rows that earlier rows do not see, and in scales."""
    page = 16

    def change(c, kb, vb, ks, vs):
        c.page = page
        odd = (0x7F, 0xFF) if kind == "f8" else (0x7FC0, 0x7F80)
        for s, n in enumerate(c.lens):
            for j in range(n, -(-n // page) * page):  # behind the end
                p, at = c.token(s, j)
                kb[p, :, at], vb[p, :, at] = odd
                if ks is not None:
                    ks[p, :, at], vs[p, :, at] = np.nan, np.inf
        p, at = c.token(0, c.lens[0] - 1)  # the last token: only the last row sees it
        vb[p, 0, at, 5] = odd[1]
        p, at = c.token(1, c.lens[1] - 2)
        kb[p, 0, at, 9] = odd[0]
        p, at = c.token(2, c.lens[2] - 3)
        vb[p, :, at] = odd[0]
        if vs is not None:
            p, at = c.token(3, c.lens[3] - 1)
            vs[p, 1, at], ks[p, 1, at] = np.nan, np.inf

    c = Case(be, [130, 95, 257, 40, 300], 4, heads, kind, page, seed=4, change=change)
    got = c.check()
    g = heads[0] // heads[1]
    assert np.isfinite(got[:3]).all() and not np.isfinite(got[3, :g, 5]).any() and np.isfinite(got[3, g:]).all()
    assert np.isfinite(got[4:6]).all() and np.isnan(got[6:8, :g]).all()
    assert np.isfinite(got[8:9]).all() and np.isnan(got[9:12]).all() and np.isfinite(got[12:15]).all() and np.isfinite(got[16:]).all()
    c.free()


def test_bad_pages_and_lengths(be):
    """Their sequences are NaN and reported; the others are right."""
    c = Case(be, [300, 40, 2000, 64, 17], 2, (4, 2, 128), seed=5)
    good = c.check()

    def with_(table=None, lens=None):
        c.be.write(c.status, np.zeros(1, np.int32))
        got = c.run(**(dict(d_pages=c.dev(table)) if table is not None else {}), **(dict(d_lens=c.dev(np.array(lens, np.int32))) if lens else {}))
        st = c.be.read(c.status, np.int32, (1,))[0]
        return got, st
    for s, i, wrong in ((0, 0, -1), (2, 77, c.cache.n_pages), (2, 124, 2 ** 31 - 1), (4, 1, -2 ** 31)):
        t = c.table.copy()
        t[s, i] = wrong
        got, st = with_(t)
        mine = np.arange(s * 2, s * 2 + 2)
        rest = np.delete(np.arange(10), mine)
        assert st == ERR_INVALID and np.isnan(got[mine]).all() and np.array_equal(got[rest], good[rest])
    for s, wrong in ((1, -1), (3, c.args["max_pages"] * 16 + 1), (0, 2 ** 31 - 1), (4, -2 ** 31)):
        lens = list(c.lens)
        lens[s] = wrong
        got, st = with_(None, lens)
        mine = np.arange(s * 2, s * 2 + 2)
        assert st == ERR_INVALID and np.isnan(got[mine]).all() and np.isfinite(np.delete(got, mine, 0)).all()
    c.be.write(c.status, np.zeros(1, np.int32))
    c.check()
    c.free()


def test_cache_past_32_bits(be):
    """Pages whose elements lie behind 2^32 bytes."""
    page, heads = 256, (8, 8, 256)
    n_pages = 2 ** 32 // (page * 8 * 256 * 2) + 3
    c = Case(be, [500, 700], 1, heads, page=page, seed=6)
    small = c.cache
    big = [be.alloc(n_pages * page * 8 * 256 * 2) for _ in range(2)]
    nbytes = page * 8 * 256 * 2
    table = c.table.copy()
    for s, n in enumerate(c.lens):
        for i in range(-(-n // page)):
            to = n_pages - 1 - (s * 4 + i)
            for a, b in zip(big, (small.d_k, small.d_v)):
                be.copy_device(be.view(a, to * nbytes, nbytes), be.view(b, int(table[s, i]) * nbytes, nbytes), nbytes)
            table[s, i] = to
    good = c.check()
    got = c.run(cache=be.kv_cache(*big, n_pages, 8, page, 256), d_pages=c.dev(table))
    assert np.array_equal(got, good)
    for b in big:
        be.free(b)
    c.free()


def test_calls_of_different_sizes_on_one_scratch(be):
    """A large call between two small ones, and the other operators of the scratch between: each the same bits."""
    a, b = Case(be, [5000, 3], 2, (16, 2, 256), seed=7), Case(be, [9, 70, 11000] * 40, 8, (8, 2, 128), "f8", seed=8)
    first = (a.run(), b.run())
    for _ in range(2):
        assert np.array_equal(a.run(), first[0]) and np.array_equal(b.run(), first[1])
    a.free(), b.free()


def test_refusals(be):
    c = Case(be, [20, 40], 2, (4, 2, 64), "f8", gate=True)
    a = c.args

    def refused(**changed):
        with pytest.raises((HipError, ValueError)) as e:
            c.run(**changed)
        assert not isinstance(e.value, HipError) or e.value.status == ERR_INVALID

    for heads in ((4, 3, 64), (4, 2, 128), (4, 4, 64), (0, 2, 64)):
        refused(heads=heads)
    for changed in (dict(rows=0), dict(rows=9), dict(n_seqs=0), dict(n_seqs=16385), dict(max_pages=0), dict(max_pages=2 ** 28), dict(scale=0.0),
                    dict(scale=float("nan")), dict(q_strides=(260, 64)), dict(q_strides=(32, 64)), dict(gate_strides=(256, 63)), dict(d_y=a["d_q"]),
                    dict(d_y=c.cache.d_v), dict(d_y=be.view(c.y, 8, c.y.nbytes - 8)), dict(d_q=be.view(a["d_q"], 2, a["d_q"].nbytes - 2))):
        refused(**changed)
    for changed in (dict(page_size=8), dict(page_size=24), dict(kv_heads=1), dict(n_pages=0), dict(d_v_scales=None),
                    dict(d_k=be.view(c.cache.d_k, 4, 64))):
        refused(cache=dataclasses.replace(c.cache, **changed))
    c.be.write(c.y, np.full(c.y.nbytes // 2, 0x1234, np.uint16))
    c.check()
    c.free()
