"""The e4m3 block-128 products on the GPU: f8_matmul and f8_experts against
their definitions in 64 bits (f8_ref.py)."""
from __future__ import annotations

import numpy as np
import pytest

import f8_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    from turboqwenfare_amd.backend import HipBackend

    with HipBackend(0) as b:
        yield b


@pytest.fixture(scope="module")
def hip():
    from turboqwenfare_amd import backend

    return backend


def bits_of(x, kind):
    return ref.to_bf16(x) if kind == "bf16" else np.ascontiguousarray(x, np.float32)


def values_of(b, kind):
    return ref.from_bf16(b) if kind == "bf16" else b


def rows_of(rng, t, n, kind):
    """Rows with a few large channels, a block of zeros and one of tiny values."""
    x = rng.standard_normal((t, n)) * np.where(rng.random(n) < 0.02, 8.0, 1.0)
    if t > 1 and n > 128:
        x[1, :128] = 0.0
        x[t - 1, 128:256] *= 2.0 ** -110
    return bits_of(x, kind)


def run_matmul(be, w, bits, kind, y_kind, offset=0):
    """The product with x and y `offset` elements into their buffers; what lies around y has to stay."""
    t, n = bits.shape
    d_x = be.to_device(np.concatenate([np.zeros(offset, bits.dtype), bits.reshape(-1), np.zeros(16, bits.dtype)]))
    guard = np.full(t * w.rows + 2 * 16 + offset, 0x4242 if y_kind == "bf16" else 7, np.uint16 if y_kind == "bf16" else np.float32)
    d_y = be.to_device(guard)
    esz = guard.itemsize
    be.f8_matmul_device(w, be.view(d_x, offset * bits.itemsize, bits.nbytes), t, be.view(d_y, (16 + offset) * esz, t * w.rows * esz),
                        x_type=kind, y_type=y_kind)
    y = be.read(d_y, guard.dtype, guard.shape)
    be.free(d_x)
    be.free(d_y)
    assert np.array_equal(y[:16 + offset], guard[:16 + offset]) and np.array_equal(y[16 + offset + t * w.rows:], guard[16 + offset + t * w.rows:])
    return values_of(y[16 + offset:16 + offset + t * w.rows], y_kind).reshape(t, w.rows).astype(np.float64)


# ---- the matrices ------------------------------------------------------------------
@pytest.mark.parametrize("rows,cols", [(1, 1), (16, 128), (33, 200), (128, 256), (130, 129), (257, 15), (512, 2048)])
def test_upload_keeps_every_byte(be, rows, cols):
    rng = np.random.default_rng(rows)
    q = rng.integers(0, 256, (rows, cols)).astype(np.uint8)
    s = rng.standard_normal((-(-rows // 128), -(-cols // 128))).astype(np.float32)
    w = be.upload_f8(q, s)
    got, scales = be.download_f8(w)
    assert np.array_equal(got, q) and np.array_equal(scales, s)
    d = be.to_device(np.concatenate([np.zeros(3, np.uint8), q.reshape(-1)]))
    d_s = be.to_device(s)
    w2 = be.upload_f8_device(be.view(d, 3, q.nbytes), d_s, rows, cols)
    got, scales = be.download_f8(w2)
    assert np.array_equal(got, q) and np.array_equal(scales, s)
    assert be.weights_bytes(w) <= be.f8_weights_bytes_for(rows, cols)
    for h in (w, w2):
        be.free_weights(h)
    for b in (d, d_s):
        be.free(b)


# ---- one matrix ----------------------------------------------------------------------
TYPES = [("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16"), ("bf16", "f32")]


def check_matmul(be, t, rows, cols, kind, y_kind, offset=0, spread=3):
    rng = np.random.default_rng(t * 7919 + rows * 31 + cols)
    q, s = ref.random_matrix(rng, rows, cols, spread)
    w = be.upload_f8(q, s)
    bits = rows_of(rng, t, cols, kind)
    got = run_matmul(be, w, bits, kind, y_kind, offset)
    want, tol = ref.matmul(values_of(bits, kind), ref.values(q, s), y_kind == "bf16" and t > 16)
    tol = tol + ref.rounding(y_kind) * (np.abs(want) + tol) + 1e-40
    worst = np.max(np.abs(got - want) / tol)
    be.free_weights(w)
    assert worst <= 1.0, (worst, np.linalg.norm(got - want) / np.linalg.norm(want))
    return np.linalg.norm(got - want) / max(np.linalg.norm(want), 1e-300)


@pytest.mark.parametrize("kind,y_kind", TYPES)
@pytest.mark.parametrize("t,rows,cols", [
    (1, 1, 1), (1, 512, 2048), (2, 17, 130), (3, 100, 100), (8, 33, 1000), (15, 48, 256), (16, 256, 2048), (16, 5, 4100), (17, 64, 128),
    (17, 1, 1), (31, 130, 300), (32, 129, 2048), (33, 257, 129), (37, 1000, 1100), (64, 300, 512), (65, 31, 640), (100, 520, 384),
    (129, 256, 1024), (200, 600, 1), (300, 777, 777)])
def test_matmul(be, t, rows, cols, kind, y_kind):
    check_matmul(be, t, rows, cols, kind, y_kind)


@pytest.mark.parametrize("kind,y_kind", TYPES)
@pytest.mark.parametrize("t", [1, 5, 40, 90])
def test_matmul_off_alignment(be, t, kind, y_kind):
    for offset, rows, cols in ((1, 64, 256), (2, 66, 250), (3, 63, 133)):
        check_matmul(be, t, rows, cols, kind, y_kind, offset=offset)


@pytest.mark.parametrize("t,rows,cols", [(1, 40000, 256), (7, 9000, 384), (16, 9001, 512), (40, 9000, 128), (1000, 40, 256)])
def test_matmul_many_rows(be, t, rows, cols):
    """Every way of dealing the weight stream to workgroups (thousands of tiles; one workgroup for all rows of x)."""
    for y_kind in ("f32", "bf16"):
        check_matmul(be, t, rows, cols, "f32", y_kind)


@pytest.mark.parametrize("kind,y_kind", TYPES)
@pytest.mark.parametrize("t,rows,cols", [
    (17, 32768, 140), (17, 32769, 140), (32, 33000, 257), (33, 33001, 129), (64, 32800, 100), (65, 32769, 130), (300, 16500, 700), (257, 40000, 77),
    (250, 65000, 300), (300, 60000, 70), (130, 33000, 450), (256, 60001, 130)])
def test_matmul_on_both_sides_of_the_split(be, t, rows, cols, kind, y_kind):
    """Matrices about as large as those from which on tiles take over from wavefronts that split K."""
    check_matmul(be, t, rows, cols, kind, y_kind)


def test_matmul_is_as_exact_as_f32(be):
    """Far from the worst case: f32 results are as near to 64 bits as random roundings of an f32 sum are (a bf16 one as its rounding)."""
    for t in (1, 16, 100):
        assert check_matmul(be, t, 300, 2048, "f32", "f32", spread=0) < 45 * 2.0 ** -24
        assert check_matmul(be, t, 300, 2048, "f32", "bf16", spread=0) < 2.0 ** -9


@pytest.mark.parametrize("y_kind", ["f32", "bf16"])
@pytest.mark.parametrize("t", [5, 16, 50, 130])
def test_a_row_that_is_no_number_is_alone(be, t, y_kind):
    rng = np.random.default_rng(t)
    q, s = ref.random_matrix(rng, 140, 300)
    w = be.upload_f8(q, s)
    x = rng.standard_normal((t, 300)).astype(np.float32)
    clean = run_matmul(be, w, x, "f32", y_kind)
    x[2, 299], x[t - 1, 7], x[1, :] = np.nan, -np.inf, np.nan
    got = run_matmul(be, w, x, "f32", y_kind)
    bad = np.isin(np.arange(t), [1, 2, t - 1])
    assert np.isnan(got[bad]).all() and np.array_equal(got[~bad], clean[~bad])
    # a NaN of the weights reaches its own output only
    q[7, 5] = 0x7F
    w2 = be.upload_f8(q, s)
    x = np.where(np.isfinite(x), x, 0).astype(np.float32)
    got = run_matmul(be, w2, x, "f32", y_kind)
    assert np.isnan(got[:, 7]).all() and np.isfinite(np.delete(got, 7, 1)).all()
    for h in (w, w2):
        be.free_weights(h)


def test_how_the_fp8_cores_cut_products(be):
    """Two products of 448 x 448 that cancel, and a small one in the same eight or another: what is left of it.  The
    tolerances for large bf16 results stand on this: at most 7 * 2^-13 of the magnitudes is lost."""
    small = np.array([448.0, 16.0, 8.0, 4.0, 1.0])
    code = [int(np.flatnonzero(ref.TABLE == v)[0]) for v in (448.0, -448.0, *small)]
    x = np.zeros((40, 128), np.float32)  # more rows than the exact path takes
    x[:, :2] = 448
    x[:, [2, 4, 7, 8, 16, 64, 127]] = 1
    for at in (2, 4, 7, 8, 16, 64, 127):
        q = np.zeros((len(small), 128), np.uint8)
        q[:, 0], q[:, 1], q[:, at] = code[0], code[1], code[2:]
        w = be.upload_f8(q, np.ones((1, 1), np.float32))
        d_x, d_y = be.to_device(ref.to_bf16(x)), be.to_device(np.zeros((40, len(small)), np.uint16))
        be.f8_matmul_device(w, d_x, 40, d_y, x_type="bf16", y_type="bf16")
        got = ref.from_bf16(be.read(d_y, np.uint16, (40, len(small))))
        # 448 = 1.75 * 2^8: the larger products count as 2^16, and 2^-13 of that is 8
        kept = np.where((small < 8) & (at < 8), 0, small)
        assert (got == kept).all() or (got == small).all(), (at, got[0])
        for b in (d_x, d_y):
            be.free(b)
        be.free_weights(w)


def test_values_at_the_borders(be):
    """Rows whose quantised values are known: ties, the largest value, subnormals, signs."""
    table = ref.TABLE[:127]
    mid = (table[1:] + table[:-1]) / 2
    cases = np.concatenate([table, mid, np.nextafter(mid, 0), np.nextafter(mid, 1e9)]).astype(np.float32)
    x = np.zeros((2 * cases.size, 128), np.float32)
    x[:, 0] = 448.0  # scale 1
    x[:cases.size, 1], x[cases.size:, 1] = cases, -cases
    q = np.zeros((2, 128), np.uint8)
    q[0, 1] = q[1, 0] = 0x38  # 1.0: the value itself, and the block's largest
    w = be.upload_f8(q, np.ones((1, 1), np.float32))
    want = ref.quantize(x)[0][:, 1]
    for part in (x, x[:16], x[100:101]):  # tiled, few rows, one row
        got = run_matmul(be, w, part, "f32", "f32")
        n = np.nonzero((x == part[0]).all(1))[0][0]
        assert np.array_equal(got[:, 0], want[n:n + len(part)]) and (got[:, 1] == 448).all()
    # the extremes of f32: a block whose largest is the largest f32, and one below 2^-100
    x = np.zeros((3, 128), np.float32)
    x[0, :2] = np.finfo(np.float32).max, 1e38
    x[1, :2] = 2.0 ** -100, 2.0 ** -103
    x[2, :2] = 2.0 ** -101, 2.0 ** -101
    got = run_matmul(be, w, x, "f32", "f32")
    qv, sv, _ = ref.quantize(x)
    assert np.allclose(got, (qv * sv)[:, [1, 0]], rtol=2.0 ** -23, atol=0) and (got[2] == 0).all()
    be.free_weights(w)


def test_matmul_large_t(be):
    """More rows than one launch dimension of a small grid, and the last rows of a long batch."""
    rng = np.random.default_rng(1)
    q, s = ref.random_matrix(rng, 24, 128)
    w = be.upload_f8(q, s)
    x = rng.standard_normal((65536, 128)).astype(np.float32)
    for y_kind in ("f32", "bf16"):
        got = run_matmul(be, w, x, "f32", y_kind)
        pick = np.r_[0:64, 32700:32800, 65472:65536]
        want, tol = ref.matmul(x[pick], ref.values(q, s), y_kind == "bf16")
        assert np.all(np.abs(got[pick] - want) <= tol + ref.rounding(y_kind) * (np.abs(want) + tol) + 1e-40)
    be.free_weights(w)


def test_matmul_refusals(be, hip):
    from turboqwenfare_amd import _lib

    q = np.zeros((32, 256), np.uint8)
    w = be.upload_f8(q, np.ones((1, 2), np.float32))
    q4 = be.synth_q4_0(64, 64, 1, 1)
    x, y = be.alloc(1 << 16), be.alloc(1 << 16)
    be.f8_matmul_device(w, x, 4, y)
    for args in ((w, x, 0, y), (w, be.view(x, 2, 8192), 2, y), (w, x, 2, be.view(y, 1, 8192)), (w, x, 4, be.view(x, 4, 8192)),
                 (hip.F8Weights(q4.handle, 32, 256), x, 2, y), (w, hip.DeviceBuffer(x.ptr, 1 << 40), 65537, hip.DeviceBuffer(y.ptr, 1 << 40))):
        with pytest.raises(hip.HipError) as e:
            be.f8_matmul_device(*args)
        assert e.value.status == _lib.ERR_INVALID
    for bad in (dict(x_type="f16"), dict(y_type="u8")):
        with pytest.raises(ValueError):
            be.f8_matmul_device(w, x, 2, y, **bad)
    with pytest.raises(ValueError):
        be.f8_matmul_device(w, x, 1000, y)
    with pytest.raises(hip.HipError):  # an F8 handle is no Q4_0 matrix, nor part of a Q4 layer
        be.q4_gemv_device(hip.Q4Weights(w.handle, 32, 256), x, 1, y)
    with pytest.raises(hip.HipError):
        be.prepare_f8_experts([w], [w], [w])  # down is not [256 x 32]
    import ctypes as C
    h = C.c_void_p()
    for rows, cols, n, ns in ((32, 256, 32 * 256 - 1, 2), (32, 256, 32 * 256, 1), (0, 256, 0, 0), (32, 0, 0, 0), (1, 65537, 65537, 513)):
        assert be.lib.tqf_hip_f8_weights_upload(be.ctx, q.ctypes.data, n, q.ctypes.data, ns, rows, cols, C.byref(h)) == _lib.ERR_INVALID
    be.free_weights(w)
    be.free_weights(q4)
    for b in (x, y):
        be.free(b)


# ---- the routed experts -----------------------------------------------------------------
class Layer:
    def __init__(self, be, n, hidden, width, seed=0):
        rng = np.random.default_rng(seed)
        self.be, self.n, self.hidden, self.width, self.handles, self.mats = be, n, hidden, width, [[], [], []], []
        for _ in range(n):
            m = [ref.random_matrix(rng, *shape, spread=1) for shape in ((width, hidden), (width, hidden), (hidden, width))]
            for i, (q, s) in enumerate(m):
                self.handles[i].append(be.upload_f8(q, s))
            self.mats.append(tuple(ref.values(q, s) for q, s in m))
        self.ex = be.prepare_f8_experts(*self.handles)

    def close(self):
        self.be.free_f8_experts(self.ex)
        for g in self.handles:
            for w in g:
                self.be.free_weights(w)

    def routes(self, rng, t, k, skew=0.0, empty=0.1):
        p = (1.0 + np.arange(self.n)) ** -skew
        ids = np.stack([rng.choice(self.n, k, replace=False, p=p / p.sum()) for _ in range(t)]).astype(np.uint16)
        w = rng.random((t, k)).astype(np.float32)
        w /= w.sum(1, keepdims=True)
        gone = rng.random((t, k)) < empty
        ids[gone] = ref.NONE
        w[gone] = np.nan  # the weight of an empty slot is not read
        return ids, w

    def run(self, bits, kind, ids, w, y_kind, offset=0):
        be, (t, n) = self.be, bits.shape
        guard = np.full(t * n + 32 + offset, 0x4242 if y_kind == "bf16" else 7, np.uint16 if y_kind == "bf16" else np.float32)
        d = [be.to_device(np.concatenate([np.zeros(offset, a.dtype), a.reshape(-1), np.zeros(8, a.dtype)])) for a in (bits, ids, w)]
        d += [be.to_device(guard), be.to_device(np.zeros(1, np.int32))]
        v = [be.view(b, offset * a.itemsize, a.nbytes) for b, a in zip(d, (bits, ids, w))]
        e = guard.itemsize
        be.f8_experts_device(self.ex, v[0], t, v[1], v[2], ids.shape[1], be.view(d[3], (16 + offset) * e, t * n * e), x_type=kind, y_type=y_kind,
                             d_status=d[4])
        y, st = be.read(d[3], guard.dtype, guard.shape), int(be.read(d[4], np.int32, (1,))[0])
        for b in d:
            be.free(b)
        assert np.array_equal(y[:16 + offset], guard[:16 + offset]) and np.array_equal(y[16 + offset + t * n:], guard[16 + offset + t * n:])
        return y[16 + offset:16 + offset + t * n].reshape(t, n), st

    def check(self, t, k, kind="f32", y_kind="f32", seed=0, skew=0.0, empty=0.1, offset=0, ids=None):
        rng = np.random.default_rng(1000 * t + k + seed)
        bits = rows_of(rng, t, self.hidden, kind)
        i, w = self.routes(rng, t, k, skew, empty)
        if ids is not None:
            i, w = ids, np.where(ids == ref.NONE, np.nan, rng.random(ids.shape)).astype(np.float32)
        got, st = self.run(bits, kind, i, w, y_kind, offset)
        assert st == 0
        got = values_of(got, y_kind).astype(np.float64)
        want, tol = ref.experts(values_of(bits, kind), i, w, self.mats, t * k > 64, y_kind)
        worst = np.max(np.abs(got - want) / (tol + 1e-35))
        assert worst <= 1.0, worst
        assert (got[(i == ref.NONE).all(1)] == 0).all()
        # On the whole the result is far nearer than that.  With e the 2-norm error of g and u, a value z of h is off by
        # about 2 e z before its rounding, which passes the middle of two steps (z / 8 at most) with a chance of that over
        # the step and then costs the step: a mean square of 2 e z * z / 8, and so sqrt(e / 4) of h and of y.  e is
        # 3.9e-5 on the fp8 cores (3.1e-3 of y) and at most 45 * 2^-24 on the others (8.2e-4); twice that is allowed.
        whole = (2.0 ** -7 if t * k > 64 else 2.0 ** -9) + (2.0 ** -8 if y_kind == "bf16" else 0)
        assert np.linalg.norm(got - want) <= whole * np.linalg.norm(want) + 1e-30
        return got


@pytest.fixture(scope="module")
def small(be):
    layer = Layer(be, 13, 384, 160)
    yield layer
    layer.close()


@pytest.fixture(scope="module")
def odd(be):
    layer = Layer(be, 5, 331, 77, 1)
    yield layer
    layer.close()


@pytest.fixture(scope="module")
def wide(be):
    layer = Layer(be, 4, 2048, 512, 2)
    yield layer
    layer.close()


@pytest.mark.parametrize("kind,y_kind", TYPES)
@pytest.mark.parametrize("t,k", [(1, 1), (1, 8), (3, 2), (8, 8), (9, 8), (13, 5), (31, 4), (37, 8), (64, 13), (100, 6), (150, 8), (301, 9)])
def test_experts(small, t, k, kind, y_kind):
    small.check(t, k, kind, y_kind)


@pytest.mark.parametrize("kind,y_kind", TYPES)
@pytest.mark.parametrize("t,k", [(1, 5), (2, 3), (12, 5), (14, 5), (50, 3), (130, 2), (200, 5)])
def test_experts_of_odd_sizes(odd, t, k, kind, y_kind):
    odd.check(t, k, kind, y_kind, offset=0)
    odd.check(t, k, kind, y_kind, offset=1)


@pytest.mark.parametrize("t,k", [(1, 4), (16, 4), (40, 4), (120, 3)])
def test_experts_of_model_width(wide, t, k):
    wide.check(t, k, "bf16", "bf16", empty=0.0)
    wide.check(t, k, "f32", "f32")


@pytest.mark.parametrize("kind,y_kind", TYPES)
@pytest.mark.parametrize("t,k", [(16, 4), (17, 3), (17, 1), (32, 2), (64, 1), (65, 1), (43, 1), (40, 1), (41, 1)])
def test_few_experts(be, t, k, kind, y_kind):
    """One and two experts: exact products up to 64 slots whatever an expert's mean, and each size of tile after them."""
    for n in (1, 2):
        layer = Layer(be, n, 200, 130, 5)
        layer.check(t, min(k, n), kind, y_kind)
        layer.close()


@pytest.mark.parametrize("t", [90, 97, 200, 700])
def test_tiles_of_one_expert(be, t):
    """One to many tiles of an expert, in numbers that do not pair, whole and not."""
    layer = Layer(be, 1, 300, 520, 6)
    for y_kind in ("f32", "bf16"):
        layer.check(t, 1, "bf16", y_kind, empty=0.0)
        layer.check(t, 1, "f32", y_kind)
    layer.close()


@pytest.mark.parametrize("t", [2, 20, 90, 400])
def test_uneven_routes(small, t):
    """One expert for every row; a popular one; the same expert in several slots; most rows empty; one row in use."""
    one = np.zeros((t, 1), np.uint16)
    small.check(t, 1, ids=one)
    small.check(t, 4, skew=2.5, empty=0.0)
    small.check(t, 3, ids=np.full((t, 3), 12, np.uint16))
    few = np.full((t, 8), ref.NONE, np.uint16)
    few[t - 1, 3] = 5
    small.check(t, 8, ids=few)
    got = small.check(t, 8, ids=np.full((t, 8), ref.NONE, np.uint16))
    assert (got == 0).all()


def test_many_experts(be):
    layer = Layer(be, 300, 64, 40, 3)
    for t, k in ((1, 16), (3, 16), (40, 16), (700, 16), (4096, 2)):
        layer.check(t, k)
    layer.close()


@pytest.mark.parametrize("t", [1, 7, 20, 200])
def test_an_expert_that_is_not_there(small, t):
    rng = np.random.default_rng(t)
    bits = rows_of(rng, t, small.hidden, "f32")
    ids, w = small.routes(rng, t, 8, empty=0.0)
    for bad in (13, 14, 1000, 0xFFFE):
        ids[t // 2, 5] = bad
        y, st = small.run(bits, "f32", ids, w, "f32")
        assert st == 1 and (y == 7).all()  # untouched
    with pytest.raises(Exception):
        small.be.f8_experts(small.ex, bits, ids, w)
    small.check(t, 8)  # and the next call is whole


@pytest.mark.parametrize("t", [4, 20, 150])
def test_rows_do_not_see_each_other(small, t):
    rng = np.random.default_rng(t)
    x = rng.standard_normal((t, small.hidden)).astype(np.float32)
    ids, w = small.routes(rng, t, 6, empty=0.0)
    clean, _ = small.run(x, "f32", ids, w, "f32")
    again, _ = small.run(x, "f32", ids, w, "f32")
    assert np.array_equal(clean, again)
    x[1, 5], x[t - 1, 0] = np.nan, np.inf
    got, _ = small.run(x, "f32", ids, w, "f32")
    rest = ~np.isin(np.arange(t), [1, t - 1])
    assert np.isnan(got[~rest]).all() and np.array_equal(got[rest], clean[rest])
    # in any order, with the same number of rows
    p = rng.permutation(t)
    shuffled, _ = small.run(np.ascontiguousarray(x[p]), "f32", np.ascontiguousarray(ids[p]), np.ascontiguousarray(w[p]), "f32")
    assert np.array_equal(shuffled, got[p], equal_nan=True)


@pytest.mark.parametrize("y_kind", ["f32", "bf16"])
@pytest.mark.parametrize("t", [5, 20, 40, 130, 400])
def test_outputs_of_very_different_sizes(be, t, y_kind):
    """Columns of one scale block that differ by 2^16, and one that is no number: each as near as it would be alone."""
    rng = np.random.default_rng(t)
    n, hidden, width, k = 3, 200, 130, 2
    mats = [[ref.random_matrix(rng, *shape, spread=1) for shape in ((width, hidden), (width, hidden), (hidden, width))] for _ in range(n)]
    for e in range(n):
        q = mats[e][2][0]
        small_rows = rng.permutation(hidden)[: hidden // 2]
        q[small_rows] = (q[small_rows] & 0x87) | 0x08  # 2^-6 and above
        q[small_rows[0]] = (q[small_rows[0]] & 0x86) | 0x78  # 2^8 and above
    mats[1][2][0][77, 5] = 0x7F  # NaN in one row of expert 1's down matrix
    layer = Layer.__new__(Layer)
    layer.be, layer.n, layer.hidden, layer.width = be, n, hidden, width
    layer.handles = [[be.upload_f8(*m[i]) for m in mats] for i in range(3)]
    layer.mats = [tuple(ref.values(*m) for m in e) for e in mats]
    layer.ex = be.prepare_f8_experts(*layer.handles)
    bits = rows_of(rng, t, hidden, "bf16")
    ids, w = layer.routes(rng, t, k)
    got, st = layer.run(bits, "bf16", ids, w, y_kind)
    assert st == 0
    got = values_of(got, y_kind).astype(np.float64)
    hit = (ids == 1).any(1)
    assert hit.any() and not hit.all()
    assert np.isnan(got[hit, 77]).all() and not np.isnan(np.delete(got[hit], 77, 1)).any() and not np.isnan(got[~hit]).any()
    layer.mats[1][2][77] = 0.0
    want, tol = ref.experts(values_of(bits, "bf16"), ids, w, layer.mats, t * k > 64, y_kind)
    # pair outputs of many rows may wait as f16: 2^-11 of each, and the sum of a row's pairs is at most the tolerance's sum
    mag = np.zeros_like(want)
    for e in range(n):
        rows, slot = np.nonzero(ids == e)
        part, _ = ref.experts(values_of(bits, "bf16")[rows], np.full((len(rows), 1), e, np.uint16), w[rows, slot][:, None], layer.mats, t * k > 64, "f32")
        np.add.at(mag, rows, np.abs(part))
    tol = tol + (2.0 ** -11 * mag if y_kind == "bf16" else 0)
    ok = np.ones_like(want, bool)
    ok[:, 77] = ~hit
    assert np.all((np.abs(got - want) <= tol + 1e-35)[ok])
    # the small columns are there, not rounded away beside the large ones: off by far less than their own size
    err = np.linalg.norm((got - want)[:, ok.all(0)], axis=0) / np.linalg.norm(want[:, ok.all(0)], axis=0)
    assert err.max() <= 2.0 ** -4, err.max()  # e4m3's half step: h's rounding may move a value by as much
    layer.close()


def test_calls_of_different_sizes_in_turn(small, odd):
    """The scratch of a large call is a smaller one's too, and another layer's."""
    for layer, t, k in ((small, 300, 8), (small, 3, 2), (odd, 100, 5), (small, 40, 8), (odd, 1, 1), (small, 300, 8)):
        layer.check(t, k, seed=t)


def test_experts_refusals(small, be, hip):
    from turboqwenfare_amd import _lib

    x, y, i, w = (be.alloc(1 << 20) for _ in range(4))
    ids = np.zeros((4, 2), np.uint16)
    be.write(i, ids)
    be.f8_experts_device(small.ex, x, 4, i, w, 2, y)
    big = lambda b: hip.DeviceBuffer(b.ptr, 1 << 40)  # noqa: E731
    for args in ((x, 0, i, w, 2, y), (big(x), 4097, big(i), big(w), 2, big(y)), (x, 4, i, w, 0, y), (x, 4, i, w, 17, y), (be.view(x, 2, 1 << 16), 4, i, w, 2, y),
                 (x, 4, be.view(i, 1, 64), w, 2, y), (x, 4, i, be.view(w, 2, 64), 2, y), (x, 4, i, w, 2, be.view(x, 8, 1 << 16))):
        with pytest.raises(hip.HipError) as e:
            be.f8_experts_device(small.ex, *args)
        assert e.value.status == _lib.ERR_INVALID
    g, u, d = small.handles
    for bad in ((g, u, g), (g, [*u[:-1], d[0]], d)):
        with pytest.raises(hip.HipError):
            be.prepare_f8_experts(*bad)
    with pytest.raises(ValueError):
        be.prepare_f8_experts(g, u[:-1], d)
    with pytest.raises(ValueError):
        be.f8_experts_device(small.ex, x, 4096, i, w, 2, y)
    for b in (x, y, i, w):
        be.free(b)


# ---- a step of a batch: router, routes, experts, head, acceptance ---------------------------
def test_experts_refuse_buffers_that_overlap_and_sizes_past_32_bits(be, small, hip):
    from turboqwenfare_amd import _lib

    n = small.hidden
    whole = be.alloc(4 * 4 * n + 4096)
    x = be.view(whole, 0, 4 * 2 * n)
    y = be.view(whole, 4 * 2 * n, 4 * 2 * n)
    ids, w = be.view(whole, 4 * 4 * n, 64), be.view(whole, 4 * 4 * n + 64, 64)
    inside = be.view(whole, 4 * 2 * n + 16, 64)
    for bad in ((x, ids, w, x), (x, inside, w, y), (x, ids, inside, y)):
        with pytest.raises(hip.HipError) as e:
            be.f8_experts_device(small.ex, bad[0], 2, bad[1], bad[2], 2, bad[3])
        assert e.value.status == _lib.ERR_INVALID
    be.free(whole)
    # one expert as wide as any: t * top_k * width of 2^32
    wide = [be.upload_f8(np.zeros(s, np.uint8), np.ones((-(-s[0] // 128), -(-s[1] // 128)), np.float32))
            for s in ((65536, 4), (65536, 4), (4, 65536))]
    ex = be.prepare_f8_experts(*([m] for m in wide))
    bufs = [be.alloc(4096 * 4 * 4), be.alloc(4096 * 16 * 2), be.alloc(4096 * 16 * 4), be.alloc(4096 * 4 * 4)]
    with pytest.raises(hip.HipError) as e:
        be.f8_experts_device(ex, bufs[0], 4096, bufs[1], bufs[2], 16, bufs[3])
    assert e.value.status == _lib.ERR_INVALID
    be.free_f8_experts(ex)
    for m in wide:
        be.free_weights(m)
    for b in bufs:
        be.free(b)


def test_a_batch_from_rows_to_tokens(be, wide):
    """Three sequences of four verify rows through the router, the experts and an F8 head on the device, then each
    sequence's acceptance: as the definitions have it, and as the host forms of the same calls."""
    rng = np.random.default_rng(11)
    seqs, k, H, V = 3, 3, wide.hidden, 1000
    t = seqs * (k + 1)
    x = rng.standard_normal((t, H)).astype(np.float32)
    router = be.upload_f32((rng.standard_normal((wide.n, H)) / 45).astype(np.float32))
    hq, hs = ref.random_matrix(rng, V, H)
    head = be.upload_f8(hq, hs * 60)
    d = {n: be.to_device(a) for n, a in dict(x=x, lg=np.zeros((t, wide.n), np.float32), ids=np.zeros((t, 2), np.uint16), w=np.zeros((t, 2), np.float32),
                                             y=np.zeros((t, H), np.float32), out=np.zeros((t, V), np.float32), st=np.zeros(1, np.int32)).items()}
    for _ in range(3):  # nothing waits between the calls, nor between the steps
        be.router_logits_device(router, d["x"], t, wide.n, H, d["lg"])
        be.route_tokens_device(d["lg"], t, wide.n, 2, d["ids"], d["w"], d_status=d["st"])
        be.f8_experts_device(wide.ex, d["x"], t, d["ids"], d["w"], 2, d["y"], d_status=d["st"])
        be.f8_matmul_device(head, d["y"], t, d["out"])
    got = {n: be.read(b, a, s) for n, b, a, s in (("lg", d["lg"], np.float32, (t, wide.n)), ("ids", d["ids"], np.uint16, (t, 2)), ("w", d["w"], np.float32, (t, 2)),
                                                  ("y", d["y"], np.float32, (t, H)), ("out", d["out"], np.float32, (t, V)))}
    assert int(be.read(d["st"], np.int32, (1,))[0]) == 0
    ids, w, _ = ref.route(got["lg"], 2)
    assert np.array_equal(got["ids"], ids) and np.allclose(got["w"], w, rtol=2.0 ** -23, atol=0)
    want, tol = ref.experts(x, ids, got["w"], wide.mats, t * 2 > 64, "f32")
    assert np.all(np.abs(got["y"] - want) <= tol)
    want, tol = ref.matmul(got["y"], ref.values(hq, hs * 60), False)
    assert np.all(np.abs(got["out"] - want) <= tol + 2.0 ** -24 * np.abs(want))
    assert np.array_equal(got["lg"], be.router_logits(router, x))
    assert np.array_equal(got["y"], be.f8_experts(wide.ex, x, ids, got["w"]))
    assert np.array_equal(got["out"], be.f8_matmul(head, got["y"]))
    import cpu_oracle as orc
    rows = (k + 1) * V * 4
    tokens = [rng.integers(0, V, k).astype(np.int32) for _ in range(seqs)]
    for s in range(seqs):
        lg = got["out"][s * (k + 1):(s + 1) * (k + 1)]
        tokens[s][:2] = lg[:2].argmax(1)  # two that a greedy target accepts
        b = [be.to_device(tokens[s]), be.alloc(4), be.alloc(4 * (k + 1))]
        be.accept_device(be.view(d["out"], s * rows, rows), None, b[0], k, V, 0.0, True, None, None, b[1], b[2])
        n = int(be.read(b[1], np.int32, (1,))[0])
        emitted = be.read(b[2], np.int32, (k + 1,))[:n + 1].tolist()
        assert (n, emitted) == orc.accept(lg, None, tokens[s], 0.0, True)
        for u in b:
            be.free(u)
    for b in d.values():
        be.free(b)
    be.free_weights(head)
    be.free_tensor(router)


def test_calls_that_share_scratch(be, small):
    """The grouped product of a Q4_0 layer and the F8 calls have one scratch: each gives the same whatever came before,
    when the scratch grows and when it does not."""
    from turboqwenfare_amd import synth

    rng = np.random.default_rng(21)
    H, F, E, own = 256, 256, 256, 24  # (a layer has 256 experts; they take turns with 24 matrices)
    mats = [(be.synth_q4_0(F, H, 3 * e, 5), be.synth_q4_0(F, H, 3 * e + 1, 5), be.synth_q4_0(H, F, 3 * e + 2, 5)) for e in range(own + 1)]
    tensors = [be.upload_f32(synth.normal((E, H), seed=1, std=H ** -0.5)), be.upload_f32(synth.normal((H,), seed=2, std=H ** -0.5))]
    layer = be.prepare_moe_layer(tensors[0], tensors[1], mats[own], *([mats[e % own][i] for e in range(E)] for i in range(3)))
    w8 = be.upload_f8(*ref.random_matrix(rng, 300, 260))
    cases = []
    for t in (3, 40, 700):
        ids, w = synth.zipf_routes(t, E, seed=t)
        cases.append(("grouped", (synth.bf16_round(synth.normal((t, H), seed=t)), ids, w)))
        ids, w = small.routes(rng, t, 8)
        cases.append(("experts", (rows_of(rng, t, small.hidden, "bf16"), ids, w)))
        cases.append(("matmul", (rng.standard_normal((t, 260)).astype(np.float32),)))

    def run(kind, args):
        if kind == "grouped":
            return be.grouped_gemm(layer, *args)
        if kind == "matmul":
            return be.f8_matmul(w8, *args)
        y, st = small.run(args[0], "bf16", args[1], args[2], "bf16")
        assert st == 0
        return y

    first = [run(*c) for c in cases]
    for at in rng.permutation(np.repeat(np.arange(len(cases)), 3)):
        assert np.array_equal(run(*cases[at]), first[at]), (cases[at][0], at)
    be.free_moe_layer(layer)
    for m in mats:
        for w in m:
            be.free_weights(w)
    for t in tensors:
        be.free_tensor(t)
    be.free_weights(w8)


def test_a_chunk_from_rows_to_logits(be):
    """A prompt chunk of bf16 rows, some of them padding (a row of masked logits), through the routes, the experts and a
    projection on the device, twice without a wait: as the definitions have it at each stage."""
    rng = np.random.default_rng(31)
    n, H, F, t, k = 12, 256, 200, 700, 4
    layer = Layer(be, n, H, F, 7)
    x = ref.to_bf16(rng.standard_normal((t, H)).astype(np.float32))
    router = (rng.standard_normal((n, H)) / 16).astype(np.float32)
    bias = rng.standard_normal(n).astype(np.float32) * 0.05
    hq, hs = ref.random_matrix(rng, 520, H)
    r, head = be.upload_f32(router), be.upload_f8(hq, hs)
    lg0 = be.to_device(np.zeros((t, n), np.float32))
    be.router_logits_device(r, be.to_device(x), t, n, H, lg0, x_type="bf16")
    lg = be.read(lg0, np.float32, (t, n))
    pad = rng.random(t) < 0.1
    lg[pad] = -np.inf
    d = {key: be.to_device(a) for key, a in dict(x=x, lg=lg, bias=bias, ids=np.zeros((t, k), np.uint16), w=np.zeros((t, k), np.float32),
                                                 y=np.zeros((t, H), np.uint16), out=np.zeros((t, 520), np.uint16), st=np.zeros(2, np.int32)).items()}
    for _ in range(2):
        be.route_tokens_device(d["lg"], t, n, k, d["ids"], d["w"], score="sigmoid", d_bias=d["bias"], n_groups=3, top_groups=2, group_best=2, scale=2.0,
                               d_status=d["st"])
        be.f8_experts_device(layer.ex, d["x"], t, d["ids"], d["w"], k, d["y"], x_type="bf16", y_type="bf16", d_status=be.view(d["st"], 4, 4))
        be.f8_matmul_device(head, d["y"], t, d["out"], x_type="bf16", y_type="bf16")
    ids, w, y, out = (be.read(d[key], a, s) for key, a, s in (("ids", np.uint16, (t, k)), ("w", np.float32, (t, k)), ("y", np.uint16, (t, H)),
                                                             ("out", np.uint16, (t, 520))))
    assert (be.read(d["st"], np.int32, (2,)) == 0).all()
    want, p, _ = ref.route(lg, k, "sigmoid", bias, 3, 2, 2, True, 2.0)
    assert np.array_equal(ids, want) and np.allclose(w, p, rtol=2.0 ** -23, atol=0) and (ids[pad] == ref.NONE).all()
    want, tol = ref.experts(values_of(x, "bf16"), ids, w, layer.mats, True, "bf16")
    part = sum(np.abs(ref.experts(values_of(x, "bf16"), ids[:, i:i + 1], w[:, i:i + 1], layer.mats, True, "f32")[0]) for i in range(k))
    got = values_of(y, "bf16").astype(np.float64)
    assert np.all(np.abs(got - want) <= tol + 2.0 ** -11 * part + 1e-35) and (got[pad] == 0).all()  # terms wait as f16
    want, tol = ref.matmul(values_of(y, "bf16"), ref.values(hq, hs), True)
    assert np.all(np.abs(values_of(out, "bf16") - want) <= tol + 2.0 ** -8 * (np.abs(want) + tol) + 1e-35)
    for b in (*d.values(), lg0):
        be.free(b)
    be.free_weights(head)
    be.free_tensor(r)
    layer.close()
