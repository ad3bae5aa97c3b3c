"""What the attention's Python calls hand to the library, and what they refuse (on the CPU)."""
from __future__ import annotations

import ctypes as C

import pytest

from turboqwenfare_amd import _lib, backend
from turboqwenfare_amd.backend import DeviceBuffer, F32Tensor, KvCache, Rope

BIG = 1 << 30


class Lib:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0
        return call


@pytest.fixture
def be():
    b = backend.HipBackend.__new__(backend.HipBackend)
    b.lib, b.ctx = Lib(), 77
    return b


def struct(arg, kind):
    return C.cast(arg, C.POINTER(kind)).contents


def buf(ptr, nbytes=BIG):
    return DeviceBuffer(ptr, nbytes)


CACHE = KvCache(buf(1 << 20), buf(2 << 20), 8, 2, 16, 64)
F8_CACHE = KvCache(buf(1 << 20), buf(2 << 20), 8, 2, 16, 64, "f8", buf(3 << 20), buf(4 << 20))


def test_rope_call(be):
    be.qk_rope_device(buf(16), buf(32), buf(48), 5, (4, 2, 64), buf(64), buf(80), d_k_out=buf(96), x_type="bf16", strides=((512, 64), None, (1024, 128)),
                      q_norm=F32Tensor(9, 64), eps=1e-5, rope=Rope(11, 32), pairs="neighbours", cache=F8_CACHE, d_slots=buf(112))
    (name, a), = be.lib.calls
    assert name == "tqf_hip_qk_rope_device" and a[0] == 77
    h, o, q, k, v = struct(a[1], _lib.Heads), struct(a[2], _lib.QkOptions), *(struct(x, _lib.HeadRows) for x in a[3:6])
    assert (h.q_heads, h.kv_heads, h.head_dim) == (4, 2, 64)
    assert (o.q_norm, o.k_norm, o.rope, o.neighbours) == (9, None, 11, 1) and abs(o.eps - 1e-5) < 1e-12
    assert [(r.data, r.row_stride, r.head_stride) for r in (q, k, v)] == [(16, 512, 64), (32, 128, 64), (48, 1024, 128)]
    assert a[6:12] == (_lib.TYPE_BF16, 5, 64, 80, 96, None) and a[13:] == (112, None)
    c = struct(a[12], _lib.KvCache)
    assert (c.d_k, c.d_v, c.d_k_scales, c.d_v_scales, c.type, c.n_pages, c.page_size, c.kv_heads, c.head_dim) == (1 << 20, 2 << 20, 3 << 20, 4 << 20,
                                                                                                               _lib.TYPE_F8, 8, 16, 2, 64)


def test_options_of_one_call_do_not_stay_for_the_next(be):
    be.qk_rope_device(buf(16), buf(32), buf(48), 5, (4, 2, 64), buf(64), buf(80), q_norm=F32Tensor(9, 64), k_norm=F32Tensor(10, 64), rope=Rope(11, 32),
                      pairs="neighbours")
    be.qk_rope_device(buf(16), buf(32), buf(48), 5, (4, 2, 64), None, buf(80))
    o = struct(be.lib.calls[1][1][2], _lib.QkOptions)
    assert (o.q_norm, o.k_norm, o.rope, o.neighbours) == (None, None, None, 0)


def test_packing_has_the_structs_layout():
    p = backend._AttnStructs
    at = lambda *path: sum(getattr(k, n).offset for k, n in path)  # noqa: E731
    o = _lib.QkOptions
    assert C.sizeof(_lib.HeadRows) == 24 and p.rows.offset == 0 and p.options.offset == 96 and p.heads.offset == 136
    assert [getattr(o, n).offset for n in ("q_norm", "k_norm", "eps", "rope", "neighbours")] == [0, 8, 16, 24, 32]
    assert [getattr(_lib.HeadRows, n).offset for n in ("data", "row_stride", "head_stride")] == [0, 8, 16]
    assert [at((p, "heads"), (_lib.Heads, n)) for n in ("q_heads", "kv_heads", "head_dim")] == [136, 140, 144]
    assert backend._ROPE_STRUCTS.size == backend._ATTN_STRUCTS.size == 148


def test_numbers_that_no_field_holds(be):
    args = buf(16), buf(32), buf(48), 5
    for heads in ((1 << 32, 2, 64), (-1, 1, 64)):
        with pytest.raises(ValueError):
            be.qk_rope_device(*args, heads, None, buf(80, 1 << 60))
    with pytest.raises(ValueError):
        be.qk_rope_device(*args, (4, 2, 64), None, buf(80), eps=1e39)
    assert be.lib.calls == []


def test_attention_calls(be):
    be.attn_prompt_device(buf(16), buf(32), buf(48), (4, 2, 64), buf(64), buf(80), 3, 10, 12, buf(96), d_gate=buf(128), gate_strides=(512, 128))
    (n1, a), = be.lib.calls
    assert n1 == "tqf_hip_attn_prompt_device" and a[2] == 0.125 and a[7:] == (64, 80, 3, 10, 12, 96, None)
    g = struct(a[6], _lib.HeadRows)
    assert (g.data, g.row_stride, g.head_stride) == (128, 512, 128)
    be.attn_paged_device(buf(16), (4, 2, 64), 3, 2, CACHE, buf(64), 4, buf(80), buf(96), scale=0.5)
    _, (n2, b) = be.lib.calls
    q, h = struct(b[3], _lib.HeadRows), struct(b[1], _lib.Heads)
    assert (q.data, q.row_stride, q.head_stride, h.q_heads, h.kv_heads, h.head_dim) == (16, 256, 64, 4, 2, 64)
    assert n2 == "tqf_hip_attn_paged_device" and b[2] == 0.5 and b[4] is None and b[5:7] == (3, 2) and b[8:] == (64, 4, 80, 96, None)


def test_small_buffers_are_refused(be):
    def refused(f, *args, **kw):
        with pytest.raises(ValueError):
            f(*args, **kw)

    rope = dict(d_q=buf(16), d_k=buf(32), d_v=buf(48), t=5, heads=(4, 2, 64), d_positions=buf(64), d_q_out=buf(80))
    row = 4 * 64
    for changed in (dict(d_q=buf(16, 4 * 5 * row - 1)), dict(d_k=buf(32, 4 * 5 * row // 2 - 4)), dict(d_q_out=buf(80, 2 * 5 * row - 2)),
                    dict(d_k_out=buf(96, 5 * row - 2)), dict(d_v_out=buf(96, 5 * row - 2)), dict(d_positions=buf(64, 16)), dict(d_slots=buf(64, 19)),
                    dict(strides=((1 << 30, 64), None, None)), dict(strides=((256, -64), None, None)), dict(x_type="f16"), dict(pairs="both")):
        refused(be.qk_rope_device, **{**rope, **changed})
    prompt = dict(d_q=buf(16), d_k=buf(32), d_v=buf(48), heads=(4, 2, 64), d_cu_q=buf(64), d_cu_k=buf(80), n_seqs=3, total_q=10, total_k=12, d_y=buf(96))
    for changed in (dict(d_q=buf(16, 20 * row - 1)), dict(d_k=buf(16, 12 * row - 1)), dict(d_v=buf(16, 12 * row - 1)), dict(d_cu_q=buf(64, 15)),
                    dict(d_cu_k=buf(64, 15)), dict(d_y=buf(96, 20 * row - 1)), dict(d_gate=buf(96, 20 * row - 1))):
        refused(be.attn_prompt_device, **{**prompt, **changed})
    paged = dict(d_q=buf(16), heads=(4, 2, 64), n_seqs=3, rows=2, cache=CACHE, d_pages=buf(64), max_pages=4, d_lens=buf(80), d_y=buf(96))
    for changed in (dict(d_q=buf(16, 12 * row - 1)), dict(d_pages=buf(64, 47)), dict(d_lens=buf(80, 11)), dict(d_y=buf(96, 12 * row - 1)),
                    dict(d_gate=buf(16, 12 * row - 1))):
        refused(be.attn_paged_device, **{**paged, **changed})
    refused(be.add_rows_device, buf(16, 39), buf(32), 10, buf(48))
    refused(be.add_rows_device, buf(16), buf(32, 39), 10, buf(48))
    refused(be.add_rows_device, buf(16), buf(32), 10, buf(48, 39))
    assert be.lib.calls == []


def test_caches(be):
    n = 8 * 2 * 16
    assert be.kv_cache(buf(16, 2 * n * 64), buf(32, 2 * n * 64), 8, 2, 16, 64).type == "bf16"
    assert be.kv_cache(buf(16, n * 64), buf(32, n * 64), 8, 2, 16, 64, "f8", buf(48, 4 * n), buf(64, 4 * n)).type == "f8"
    for bad in ((buf(16, 2 * n * 64 - 1), buf(32), 8, 2, 16, 64), (buf(16), buf(32, 2 * n * 64 - 1), 8, 2, 16, 64), (buf(16), buf(32), 8, 2, 16, 64, "f8"),
                (buf(16), buf(32), 8, 2, 16, 64, "f8", buf(48), buf(64, 4 * n - 1)), (buf(16), buf(32), 8, 2, 16, 64, "f32")):
        with pytest.raises(ValueError):
            be.kv_cache(*bad)


def test_frequencies(be):
    with pytest.raises(ValueError):
        be.prepare_rope([[1.0, 2.0]])
