"""Attention of packed prompts on the GPU against its definition in 64 bits (attn_ref.py), and what it refuses."""
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


def bf16(x):
    bits = f8_ref.to_bf16(np.ascontiguousarray(x, np.float32))
    return bits, f8_ref.from_bf16(bits).astype(np.float64)


class Case:
    """Sequences of (queries, keys); rows between and around the parts of a wider buffer, guards behind y."""

    def __init__(self, be, seqs, heads, gate=False, seed=0, gaps=(0, 0, 0, 0), behind=(0, 0), sharp=1.0, change=None):
        self.be, self.heads, self.seqs = be, heads, seqs
        nq, nk, d = heads
        rng = np.random.default_rng(seed)
        self.cu_q = np.concatenate([[0], np.cumsum([s[0] for s in seqs])]).astype(np.int32)
        self.cu_k = np.concatenate([[0], np.cumsum([s[1] for s in seqs])]).astype(np.int32)
        tq, tk = int(self.cu_q[-1]) + behind[0], int(self.cu_k[-1]) + behind[1]
        self.tq, self.tk = tq, tk
        x = [rng.standard_normal((t, n, d + g)) for t, n, g in zip((tq, tk, tk, tq), (nq, nk, nk, nq), gaps)]
        x[0] *= sharp
        if change:
            change(self, x)
        both = [bf16(a) for a in x]
        self.q, self.k, self.v, g64 = [b[1][..., :d] for b in both]
        self.gate = g64 if gate else None
        self.keep = []
        dev = self.dev
        bufs = [dev(b[0]) if b[0].size else dev(np.zeros(8, np.uint16)) for b in both]
        strides = [(n * (d + g), d + g) for n, g in zip((nq, nk, nk, nq), gaps)]
        self.y = dev(np.full(tq * nq * d + 8, 0x1234, np.uint16))
        self.status = dev(np.zeros(1, np.int32))
        self.args = dict(d_q=bufs[0], d_k=bufs[1], d_v=bufs[2], heads=heads, d_cu_q=dev(self.cu_q), d_cu_k=dev(self.cu_k), n_seqs=len(seqs),
                         total_q=tq, total_k=tk, d_y=self.y, strides=tuple(strides[:3]), d_status=self.status,
                         **(dict(d_gate=bufs[3], gate_strides=strides[3]) if gate else {}))

    def dev(self, a):
        self.keep.append(self.be.to_device(a))
        return self.keep[-1]

    def run(self, **changed):
        self.be.attn_prompt_device(**{**self.args, **changed})
        nq, _, d = self.heads
        raw = self.be.read(self.y, np.uint16, (self.tq * nq * d + 8,))
        assert (raw[-8:] == 0x1234).all()
        self.raw = raw[:-8].reshape(self.tq, nq, d)
        return f8_ref.from_bf16(self.raw).astype(np.float64)

    def check(self, scale=None, **changed):
        s = self.heads[2] ** -0.5 if scale is None else scale
        got = self.run(scale=scale, **changed)
        want, tol = ref.prompt(self.q, self.k, self.v, self.cu_q, self.cu_k, s, self.gate)
        out = np.isnan(tol)
        assert (self.raw[self.cu_q[-1]:] == 0x1234).all()  # rows behind the last sequence
        same = (np.isnan(got) & np.isnan(want)) | (got == want)
        bad = ~(np.abs(got - want) <= tol) & ~same & ~out
        assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], tol[bad][:5])
        assert self.be.read(self.status, np.int32, (1,))[0] == 0
        return got

    def free(self):
        for b in self.keep:
            self.be.free(b)


HEADS = [(16, 2, 256), (8, 2, 128), (4, 4, 64), (6, 2, 64), (7, 1, 128), (1, 1, 256), (3, 3, 128), (8, 1, 64)]


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("n", [1, 2, 31, 33, 64, 65, 127, 200])
def test_one_prompt(be, heads, n):
    c = Case(be, [(n, n)], heads, gate=n % 2 == 0, seed=n)
    c.check()
    c.free()


@pytest.mark.parametrize("heads", HEADS)
def test_packed(be, heads):
    """Lengths of 0, 1 and more, chunks with earlier keys, sequences without keys or with fewer than queries, rows behind all."""
    c = Case(be, [(5, 5), (0, 0), (1, 1), (70, 130), (0, 9), (33, 0), (40, 7), (129, 129), (1, 300), (64, 64), (3, 66)], heads, gate=True,
             seed=3, gaps=(8, 0, 16, 8), behind=(9, 5))
    c.check()
    got = c.run()
    assert (got[c.cu_q[5]:c.cu_q[6]] == 0).all()  # no keys
    assert (got[c.cu_q[6]:c.cu_q[6] + 33] == 0).all()  # queries in front of the first key
    c.free()


@pytest.mark.parametrize("heads", [(16, 2, 256), (8, 4, 128), (4, 2, 64)])
def test_longer(be, heads):
    c = Case(be, [(300, 1500), (700, 700), (1, 2049)], heads, seed=4)
    c.check()
    c.free()


@pytest.mark.parametrize("heads", [(2, 1, 256), (2, 1, 128), (2, 1, 64)])
def test_sharp_and_flat_softmax(be, heads):
    """Scores of hundreds (weights of one key), maxima that grow late, and all alike."""
    def late(c, x):
        x[1] *= np.linspace(0.1, 3.0, x[1].shape[0])[:, None, None]
    for sharp, change in ((40.0, None), (0.0, None), (12.0, late)):
        c = Case(be, [(190, 190), (37, 260)], heads, seed=5, sharp=sharp, change=change)
        c.check()
        c.check(scale=0.9)
        c.check(scale=1e-3)
        c.free()


@pytest.mark.parametrize("heads", [(4, 2, 256), (4, 2, 128), (4, 2, 64)])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
def test_odd_values_stay_with_the_rows_that_see_them(be, heads, what):
    """An infinity or a NaN in a value, a key, or behind a sequence does not reach rows that do not see it."""
    def change(c, x):
        k, v = x[1], x[2]
        a = c.cu_k
        v[a[0] + 50, 0, 3] = what      # rows 50.. of sequence 0 see it
        v[a[0] + 120, 1, 7:40] = what
        k[a[1] + 20, 0, 5] = np.nan    # rows 20.. of sequence 1
        v[a[2] + 0, 0, 1] = what       # all of sequence 2
        k[c.cu_k[-1]:], v[c.cu_k[-1]:] = np.nan, what  # behind all
        k[a[4]:a[5]], v[a[4]:a[5]] = np.nan, np.nan  # a sequence without queries, between others
    c = Case(be, [(150, 150), (70, 70), (40, 90), (45, 45), (0, 40), (64, 64)], heads, seed=6, behind=(0, 30), change=change)
    got = c.check()
    assert np.isfinite(got[:50]).all() and not np.isfinite(got[50:150, :2, 3]).any() and np.isfinite(got[c.cu_q[3]:]).all()
    c.free()


def test_both_infinities(be):
    """+inf and -inf in one column are NaN from the second on; a row's other columns stay."""
    def change(c, x):
        x[2][10, 0, 4], x[2][20, 0, 4] = np.inf, -np.inf
    c = Case(be, [(40, 40)], (2, 1, 128), seed=7, change=change)
    got = c.check()
    assert np.isfinite(got[:10]).all() and np.isposinf(got[10:20, :, 4]).all() and np.isnan(got[20:, :, 4]).all()
    c.free()


def test_a_key_further_on_changes_nothing(be):
    """Bit by bit: rows in front of a change of later keys and values."""
    def change(c, x):
        x[1][90:], x[2][90:] = 5.0, -7.0
    a, b = Case(be, [(200, 200)], (8, 2, 128), seed=8), Case(be, [(200, 200)], (8, 2, 128), seed=8, change=change)
    a.run(), b.run()
    assert np.array_equal(a.raw[:90], b.raw[:90]) and not np.array_equal(a.raw[90:], b.raw[90:])
    a.free(), b.free()


def test_many_sequences(be):
    """More than a wavefront looks through at once, most of a row or two."""
    seqs = [(1 + i % 3, 1 + i % 3 + i % 5) for i in range(300)]
    c = Case(be, seqs, (4, 2, 64), seed=9)
    c.check()
    c.free()


def test_bounds_out_of_range_are_reported(be):
    c = Case(be, [(20, 20), (30, 30)], (2, 1, 64), seed=10, behind=(4, 4))
    for cu_q, cu_k in (([0, 20, 60], [0, 20, 50]), ([0, 20, 50], [0, 20, 2 ** 31 - 1]), ([0, -1, 50], [0, 20, 50]), ([0, 20, 10], [0, 20, 50]),
                       ([-5, 20, 50], [0, 20, 50]), ([0, 20, 50], [0, 55, 50])):
        c.be.write(c.status, np.zeros(1, np.int32))
        c.run(d_cu_q=c.dev(np.array(cu_q, np.int32)), d_cu_k=c.dev(np.array(cu_k, np.int32)))
        assert c.be.read(c.status, np.int32, (1,))[0] == ERR_INVALID
    c.be.write(c.status, np.zeros(1, np.int32))
    c.be.write(c.y, np.full(c.y.nbytes // 2, 0x1234, np.uint16))
    c.check()
    c.free()


def test_no_keys_at_all(be):
    c = Case(be, [(5, 0), (3, 0)], (2, 1, 128), seed=11)
    assert c.tk == 0 and (c.check() == 0).all()
    c.free()


def test_refusals(be):
    c = Case(be, [(8, 8)], (4, 2, 64), gate=True)
    a = c.args

    def refused(**changed):
        with pytest.raises((HipError, ValueError)) as e:
            c.run(**changed)
        assert not isinstance(e.value, HipError) or e.value.status == ERR_INVALID

    for heads in ((4, 3, 64), (4, 2, 32), (0, 1, 64), (258, 2, 64)):
        refused(heads=heads)
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        refused(scale=scale)
    for changed in (dict(n_seqs=0), dict(n_seqs=16385), dict(total_q=0), dict(total_q=2 ** 20 + 1), dict(total_k=2 ** 31)):
        refused(**changed)
    refused(strides=((260, 64), (128, 64), (128, 64)))
    refused(strides=((256, 64), (128, 60), (128, 64)))
    refused(strides=((256, 64), (128, 64), (32, 64)))
    refused(strides=((256, 64), (128, 64), (2 ** 24, 64)))
    refused(gate_strides=(258, 64))
    refused(d_q=be.view(a["d_q"], 2, a["d_q"].nbytes - 2))
    refused(d_v=be.view(a["d_v"], 8, a["d_v"].nbytes - 8))
    refused(d_y=a["d_q"])
    refused(d_y=a["d_gate"])
    refused(d_y=be.view(c.y, 8, c.y.nbytes - 8))
    refused(d_y=be.view(c.y, 0, 16))
    c.be.write(c.y, np.full(c.y.nbytes // 2, 0x1234, np.uint16))
    c.check()
    c.free()
