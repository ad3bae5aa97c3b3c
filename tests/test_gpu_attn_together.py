"""The attention's calls one after another, on two streams at once, and far apart in memory."""
from __future__ import annotations

import numpy as np
import pytest

import attn_ref as ref
import f8_ref
from test_gpu_attn_prompt import Case, be, bf16  # noqa: F401
from turboqwenfare_amd import _lib

pytestmark = pytest.mark.gpu


class Sequence:
    """Projections [t, q_heads + 2 kv_heads, d] of one sequence, and a cache for it."""

    def __init__(self, be, heads, t, page=16, kind="bf16", seed=0):  # noqa: F811
        self.be, self.heads, self.t, self.page = be, heads, t, page
        nq, nk, d = heads
        rng = np.random.default_rng(seed)
        bits, self.x = bf16(rng.standard_normal((t, nq + 2 * nk, d)))
        self.pages = -(-t // page) + 1
        self.table = rng.permutation(self.pages).astype(np.int32)
        at = np.arange(t)
        self.freq = 1e4 ** (-np.arange(d // 4) / (d // 4))
        self.rope, self.cache = be.prepare_rope(self.freq), be.alloc_kv_cache(self.pages, nk, page, d, kind)
        self.keep = []
        dev = lambda a: self.keep.append(be.to_device(a)) or self.keep[-1]  # noqa: E731
        self.rows, self.positions, self.d_table = dev(bits), dev(at.astype(np.int32)), dev(self.table)
        self.slots = dev((self.table[at // page] * page + at % page).astype(np.int32))
        self.q, self.k, self.y = (dev(np.zeros((t, n, d), np.uint16)) for n in (nq, nk, nq))
        self.status, self.dev = dev(np.zeros(1, np.int32)), dev

    def rotate(self, first, n):
        be, (nq, nk, d) = self.be, self.heads
        row = (nq + 2 * nk) * d
        part = lambda h: be.view(self.rows, 2 * (first * row + h * d), self.rows.nbytes - 2 * (first * row + h * d))  # noqa: E731
        out = lambda b, heads: be.view(b, 2 * first * heads * d, 2 * n * heads * d)  # noqa: E731
        be.qk_rope_device(part(0), part(nq), part(nq + nk), n, self.heads, be.view(self.positions, 4 * first, 4 * n), out(self.q, nq),
                          d_k_out=out(self.k, nk), x_type="bf16", strides=((row, d),) * 3, rope=self.rope, cache=self.cache,
                          d_slots=be.view(self.slots, 4 * first, 4 * n), d_status=self.status)

    def prompt(self, first, n):
        """Rows first.. before which there are others: keys as the rotation left them, values where the projection put them."""
        be, (nq, nk, d) = self.be, self.heads
        row = (nq + 2 * nk) * d
        be.attn_prompt_device(be.view(self.q, 2 * first * nq * d, 2 * n * nq * d), self.k, be.view(self.rows, 2 * (nq + nk) * d, self.rows.nbytes - 2 * (nq + nk) * d),
                              self.heads, self.dev(np.array([0, n], np.int32)), self.dev(np.array([0, first + n], np.int32)), 1, n, first + n,
                              be.view(self.y, 2 * first * nq * d, 2 * n * nq * d), strides=(None, None, (row, d)), d_status=self.status)

    def verify(self, first, n):
        be, (nq, _, d) = self.be, self.heads
        be.attn_paged_device(be.view(self.q, 2 * first * nq * d, 2 * n * nq * d), self.heads, 1, n, self.cache, self.d_table, self.pages,
                             self.dev(np.array([first + n], np.int32)), be.view(self.y, 2 * first * nq * d, 2 * n * nq * d), d_status=self.status)

    def check(self):
        be, (nq, nk, d) = self.be, self.heads
        q = f8_ref.from_bf16(be.read(self.q, np.uint16, (self.t, nq, d))).astype(np.float64)
        k = f8_ref.from_bf16(be.read(self.k, np.uint16, (self.t, nk, d))).astype(np.float64)
        want, tol = ref.attention(q, k, self.x[:, nq + nk:], np.arange(self.t), d ** -0.5)
        got = f8_ref.from_bf16(be.read(self.y, np.uint16, (self.t, nq, d))).astype(np.float64)
        assert (np.abs(got - want) <= tol).all()
        assert be.read(self.status, np.int32, (1,))[0] == 0
        return got

    def free(self):
        for b in self.keep:
            self.be.free(b)
        self.be.free_kv_cache(self.cache)
        self.be.free_rope(self.rope)


@pytest.mark.parametrize("heads", [(16, 2, 256), (8, 2, 128), (3, 1, 64)])
def test_a_prompt_in_chunks_and_then_tokens(be, heads):  # noqa: F811
    """Every row of a sequence, whichever call made it, against the whole sequence's definition."""
    s = Sequence(be, heads, 1337)
    at = 0
    for n in (1, 300, 37, 911):
        s.rotate(at, n), s.prompt(at, n)
        at += n
    for n in (1, 8, 3, 1, 5, 7, 2):
        s.rotate(at, n), s.verify(at, n)
        at += n
    while at < s.t:
        n = min(8, s.t - at)
        s.rotate(at, n), s.verify(at, n)
        at += n
    s.check()
    s.free()


def test_drafts_that_are_not_accepted_leave_nothing(be):  # noqa: F811
    """Rows written behind the sequence and then over: bit for bit what a sequence without them gives."""
    a, b = Sequence(be, (8, 2, 128), 200, seed=5), Sequence(be, (8, 2, 128), 200, seed=5)
    for s in (a, b):
        s.rotate(0, 100), s.prompt(0, 100)
    for at in range(100, 200, 4):
        n = min(8, 200 - at)
        a.rotate(at, n), a.verify(at, n)  # up to eight, of which four stay
        a.rotate(at, 4), a.verify(at, 4)
        b.rotate(at, 4), b.verify(at, 4)
    assert np.array_equal(a.check(), b.check())
    a.free(), b.free()


def test_two_streams_at_once():
    """Two contexts with calls under way at the same time, each with workspaces of its own."""
    from turboqwenfare_amd.backend import HipBackend

    with HipBackend(0) as one, HipBackend(0) as two:
        seqs = [Sequence(one, (16, 2, 256), 700, seed=6), Sequence(two, (8, 2, 128), 700, seed=7)]
        for at in range(0, 700, 100):
            for s in seqs:
                s.rotate(at, 100), s.prompt(at, 100)
            for s in seqs:
                for i in range(92, 100, 4):  # and the last rows once more, over the cache
                    s.verify(at + i, 4)
        for s in seqs:
            s.check()
            s.free()


def test_the_same_call_gives_the_same_bits(be):  # noqa: F811
    c = Case(be, [(40, 3000), (500, 500), (1, 2000)], (16, 2, 256), gate=True, seed=8)
    c.run()
    first = c.raw.copy()
    for _ in range(4):
        c.run()
        assert np.array_equal(c.raw, first)
    c.free()


@pytest.mark.parametrize("parts", [False, True])
def test_keys_past_32_bits(be, parts):  # noqa: F811
    """Rows of keys and values 2^22 elements apart: the last ones are past 2^32 bytes and 2^31 elements."""
    nq, nk, d, n, row = 4, 2, 64, 640, 1 << 22
    lq = 40 if parts else n
    rng = np.random.default_rng(9)
    (qb, q), (kb, k), (vb, v) = (bf16(rng.standard_normal((t, h, d))) for t, h in ((lq, nq), (n, nk), (n, nk)))
    far = be.alloc(2 * n * row)
    for t in range(n):
        be.write(be.view(far, 2 * t * row, 2 * nk * d), kb[t])
        be.write(be.view(far, 2 * (t * row + 4096), 2 * nk * d), vb[t])
    bufs = [be.to_device(x) for x in (qb, np.array([0, lq], np.int32), np.array([0, n], np.int32), np.zeros((lq, nq, d), np.uint16))]
    be.attn_prompt_device(bufs[0], far, be.view(far, 8192, far.nbytes - 8192), (nq, nk, d), bufs[1], bufs[2], 1, lq, n, bufs[3],
                          strides=(None, (row, d), (row, d)))
    got = f8_ref.from_bf16(be.read(bufs[3], np.uint16, (lq, nq, d))).astype(np.float64)
    want, tol = ref.attention(q, k, v, np.arange(lq) + n - lq, d ** -0.5)
    assert (np.abs(got - want) <= tol).all()
    for b in (*bufs, far):
        be.free(b)


def test_kernels_are_counted(be):  # noqa: F811
    s = Sequence(be, (4, 2, 64), 50, seed=10)
    be.profile_enable(True)
    try:
        s.rotate(0, 40), s.prompt(0, 40), s.rotate(40, 10), s.verify(42, 8)
        counts = [be.profile_read(k) for k in (_lib.KERNEL_QK_ROPE, _lib.KERNEL_ATTN_PROMPT, _lib.KERNEL_ATTN_PAGED)]
    finally:
        be.profile_enable(False)
    assert [c[0] for c in counts] == [2, 1, 1] and all(c[1] > 0 for c in counts)
    s.free()


def test_other_calls_on_the_same_workspace(be):  # noqa: F811
    """Between the attention's calls the workspace is another operator's."""
    rng = np.random.default_rng(11)
    w = be.upload_f8(*f8_ref.random_matrix(rng, 256, 512))
    x = rng.standard_normal((700, 512)).astype(np.float32)
    want = be.f8_matmul(w, x)
    c = Case(be, [(33, 2500)], (16, 2, 256), seed=12)
    first = c.check()
    for _ in range(3):
        assert np.array_equal(be.f8_matmul(w, x), want)
        assert np.array_equal(c.run(), first)
    be.free_weights(w)
    c.free()
