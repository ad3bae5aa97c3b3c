"""Attention over the cache where sequences are cut into many parts, and parts have many sequences: with keys of which none
can be left out or counted twice unseen (attn_marks.py), against the definition in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

import attn_marks as marks
import f8_ref
from test_gpu_attn_paged import Case, be, bf16  # noqa: F401

pytestmark = pytest.mark.gpu

UP_AND_DOWN = pytest.mark.parametrize("ramp", [0, 1, 2], ids=["flat", "up", "down"])
KINDS = pytest.mark.parametrize("kind", ["bf16", "f8"])


def marked(be, lens, rows, heads, kind, page, ramp, seed=0, odd=None, **kw):  # noqa: F811
    nk, d = heads[1:]

    def change(c, kb, vb, ks, vs):
        c.page = page
        rng = np.random.default_rng(seed + 1)
        for s, n in enumerate(c.lens):
            k, v = marks.keys_and_values(rng, n, nk, d, marks.RAMPS[kind][ramp])
            j = np.arange(n)
            p, at = c.table[s, j // page], j % page
            if kind == "f8":
                kb[p, :, at], ks[p, :, at], _ = marks.e4m3(k)
                vb[p, :, at], vs[p, :, at], _ = marks.e4m3(v)
            else:
                kb[p, :, at], vb[p, :, at] = bf16(k)[0], bf16(v)[0]
        if odd:
            odd(c, kb, vb, ks, vs)

    c = Case(be, lens, rows, heads, kind, page, seed=seed, change=change, **kw)
    bits, c.q = bf16(marks.queries(c.q))
    c.args["d_q"] = c.dev(bits)
    return c


def mixed(n, most, seed):
    """Lengths of 0 to `most`, the short ones as frequent as the long."""
    rng = np.random.default_rng(seed)
    lens = np.exp(rng.uniform(0, np.log(most), n)).astype(int)
    lens[rng.integers(0, n, 2)] = 0
    lens[rng.integers(0, n, 2)] = most
    return lens.tolist()


@KINDS
@UP_AND_DOWN
@pytest.mark.parametrize("heads", [(16, 2, 256), (8, 2, 128), (2, 2, 64)])
def test_long(be, kind, ramp, heads):  # noqa: F811
    """Cut into many parts, beside short ones."""
    c = marked(be, [9000, 40, 20000, 1], 2, heads, kind, 16, ramp, seed=2)
    c.check()
    c.free()


@KINDS
@UP_AND_DOWN
@pytest.mark.parametrize("heads, rows", [((2, 1, 256), 1), ((4, 1, 128), 8), ((1, 1, 64), 4)])
def test_one_long(be, kind, ramp, heads, rows):  # noqa: F811
    """One sequence, a step or two to a workgroup."""
    c = marked(be, [19999], rows, heads, kind, 32, ramp, seed=3)
    c.check()
    c.free()


@KINDS
@UP_AND_DOWN
@pytest.mark.parametrize("heads, rows", [((16, 2, 256), 4), ((16, 2, 256), 8), ((8, 2, 256), 3), ((16, 2, 128), 4), ((32, 4, 64), 4)])
def test_verify_rows_of_many_sequences(be, kind, ramp, heads, rows):  # noqa: F811
    """More steps than workgroups: each has several, and the ends of some sequences beside the beginnings of others.  Two
    tiles of rows, and (8 rows) two workgroups for the rows of a key head."""
    c = marked(be, mixed(48, 3000, rows), rows, heads, kind, 16, ramp, seed=4, gate=True)
    c.check()
    c.free()


@KINDS
@UP_AND_DOWN
@pytest.mark.parametrize("heads, rows", [((32, 1, 128), 8), ((24, 1, 256), 8), ((20, 1, 64), 7)])
def test_many_rows_of_a_key_head(be, kind, ramp, heads, rows):  # noqa: F811
    """Several workgroups for the rows of a part, which has several sequences."""
    c = marked(be, mixed(64, 3000, rows), rows, heads, kind, 32, ramp, seed=5)
    c.check()
    c.free()


@KINDS
@UP_AND_DOWN
@pytest.mark.parametrize("heads, rows, n", [((8, 8, 128), 1, 80), ((8, 2, 256), 1, 150), ((16, 2, 256), 4, 150), ((16, 4, 128), 8, 160), ((8, 8, 64), 2, 150)])
def test_more_heads_than_workgroups(be, kind, ramp, heads, rows, n):  # noqa: F811
    """More (sequence, key head) than parts, so that cuts are kept by part."""
    c = marked(be, mixed(n, 700, n), rows, heads, kind, 16, ramp, seed=6)
    c.check()
    c.free()


@KINDS
@pytest.mark.parametrize("heads, rows", [((16, 2, 256), 4), ((16, 2, 256), 8), ((8, 2, 128), 4), ((4, 2, 64), 6), ((16, 1, 128), 8)])
def test_odd_values_in_drafts_of_many_sequences(be, kind, heads, rows):  # noqa: F811
    """NaN and infinities in the last tokens of every third sequence, which only some of its rows see: the others, and the
    sequences that the same workgroups go on with, have none of them."""
    lens = [n + rows for n in mixed(48, 3000, 7)]

    def odd(c, kb, vb, ks, vs):
        what = (0x7F, 0xFF) if kind == "f8" else (0x7FC0, 0x7F80)
        for s in range(0, len(lens), 3):
            p, at = c.token(s, lens[s] - 1 - s % (rows - 1))
            vb[p, 0, at, s % 64] = what[s % 2]
            if s % 2:
                kb[p, 1 % heads[1], at, 5] = what[0]
            elif vs is not None:
                vs[p, :, at] = np.inf

    c = marked(be, lens, rows, heads, kind, 16, 0, seed=8, odd=odd)
    got = c.check().reshape(len(lens), rows, *heads[::2])
    for s in range(len(lens)):
        first = rows if s % 3 else rows - 1 - s % (rows - 1)  # the first row that sees an odd one
        assert np.isfinite(got[s, :first]).all() and not (s % 3 == 0 and np.isfinite(got[s, first:, 0]).all())
    c.free()


@KINDS
def test_bad_pages_among_many_sequences(be, kind):  # noqa: F811
    """Their rows alone are NaN, with several sequences to a workgroup."""
    heads, rows = (16, 2, 256), 4
    lens = [n + 1 for n in mixed(48, 2000, 9)]
    c = marked(be, lens, rows, heads, kind, 16, 1, seed=9)
    good = c.check()
    table = c.table.copy()
    bad = list(range(0, 48, 5))
    for s in bad:
        table[s, (lens[s] - 1) // 16 * (s % 2)] = [-1, c.cache.n_pages][s % 2]
    got = c.run(d_pages=c.dev(table)).reshape(48, rows, -1)
    rest = np.delete(np.arange(48), bad)
    assert np.isnan(got[bad]).all() and np.array_equal(got[rest], good.reshape(48, rows, -1)[rest])
    assert c.be.read(c.status, np.int32, (1,))[0] != 0
    c.free()
