"""Routes of the batched router as the routes of a Q4_0 layer's grouped product, and what the profile counts of F8 calls."""
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


@pytest.mark.parametrize("t", [1, 37, 700])
def test_routes_feed_the_grouped_product(be, t):
    """Rows through router_logits_device, route_tokens_device (softmax, top 8, renormalised) and grouped_gemm_device without
    a wait: the host forms' results for routes that the definition gives."""
    from turboqwenfare_amd import synth

    H, F, E, own = 256, 256, 256, 24  # (the 256 experts take turns with 24 matrices)
    mats = [(be.synth_q4_0(F, H, 3 * e, 5), be.synth_q4_0(F, H, 3 * e + 1, 5), be.synth_q4_0(H, F, 3 * e + 2, 5)) for e in range(own + 1)]
    router, shared = be.upload_f32(synth.normal((E, H), seed=1, std=H ** -0.5)), be.upload_f32(synth.normal((H,), seed=2, std=H ** -0.5))
    layer = be.prepare_moe_layer(router, shared, mats[own], *([mats[e % own][i] for e in range(E)] for i in range(3)))
    x = synth.bf16_round(synth.normal((t, H), seed=t))
    d = {n: be.to_device(a) for n, a in dict(x=x, lg=np.zeros((t, E), np.float32), ids=np.zeros((t, 8), np.uint16), w=np.zeros((t, 8), np.float32),
                                             y=np.zeros((t, H), np.float32), st=np.zeros(2, np.int32)).items()}
    for _ in range(2):
        be.router_logits_device(router, d["x"], t, E, H, d["lg"], x_type="bf16")
        be.route_tokens_device(d["lg"], t, E, 8, d["ids"], d["w"], d_status=d["st"])
        be.grouped_gemm_device(layer, d["x"], t, d["ids"], d["w"], d["y"], be.view(d["st"], 4, 4))
    lg, ids, w, y, st = (be.read(d[n], a, s) for n, a, s in (("lg", np.float32, (t, E)), ("ids", np.uint16, (t, 8)), ("w", np.float32, (t, 8)),
                                                            ("y", np.float32, (t, H)), ("st", np.int32, (2,))))
    assert (st == 0).all()
    want, p, _ = ref.route(lg, 8)
    assert np.array_equal(ids, want) and np.all(np.abs(w - p) <= 2.0 ** -24 * p * (1 + 1e-6))
    assert np.array_equal(y, be.grouped_gemm(layer, x, want, w)) and np.abs(y).max() > 0
    for b in d.values():
        be.free(b)
    be.free_moe_layer(layer)
    for m in mats:
        for h in m:
            be.free_weights(h)
    for h in (router, shared):
        be.free_tensor(h)


def test_profile_of_f8_calls(be):
    """A product's and a router's bytes are those of its operands; the experts' are left to the caller, who has the ids."""
    from turboqwenfare_amd import _lib

    rng = np.random.default_rng(0)
    q, s = ref.random_matrix(rng, 300, 260)
    w, r = be.upload_f8(q, s), be.upload_f32(np.zeros((16, 260), np.float32))
    m = [be.upload_f8(*ref.random_matrix(rng, *shape)) for shape in ((64, 260), (64, 260), (260, 64))]
    ex = be.prepare_f8_experts(*([h] for h in m))
    x = rng.standard_normal((40, 260)).astype(np.float32)
    be.profile_enable()
    be.f8_matmul(w, x)
    be.router_logits(r, x)
    be.route_tokens(np.zeros((40, 16), np.float32), 2)
    be.f8_experts(ex, x, np.zeros((40, 1), np.uint16), np.ones((40, 1), np.float32))
    n, ms, by = be.profile_read(_lib.KERNEL_F8_MATMUL)
    assert n == 1 and ms > 0 and by == 4 * 40 * (260 + 300) + 300 * 260 + 4 * 9
    n, ms, by = be.profile_read(_lib.KERNEL_ROUTER)
    assert n == 2 and ms > 0 and by == 4 * (40 * 260 + 16 * 260 + 40 * 16) + 4 * 40 * 16 + 6 * 40 * 2
    n, ms, by = be.profile_read(_lib.KERNEL_F8_EXPERTS)
    assert n == 1 and ms > 0 and by == 0
    be.profile_enable(False)
    be.free_f8_experts(ex)
    for h in (w, *m):
        be.free_weights(h)
    be.free_tensor(r)
