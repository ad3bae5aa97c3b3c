"""The MTP loop with attention layers in the target: every stage of every pass replayed in 64 bits from the device's own
inputs to it, positions and caches followed through drafts that are accepted and that are not."""
from __future__ import annotations

import numpy as np
import pytest

import attn_ref as ref
import cpu_oracle as orc
import f8_ref
from conftest import rel_err
from stack_oracle import oracle_replay
from turboqwenfare_amd.mtp_loop import DeviceEngine, MtpLoop, MtpModel
from turboqwenfare_amd.workloads import H

pytestmark = pytest.mark.gpu

LAYERS, VOCAB, K, T = 2, 32768, 3, 0.7
KINDS = {
    "gated_256": dict(heads=(16, 2, 256), rotary=64, max_tokens=200, page=16),
    "plain_128_f8": dict(heads=(8, 8, 128), rotary=128, gated=False, max_tokens=150, page=32, cache="f8"),
}


@pytest.fixture(scope="module", params=list(KINDS))
def model(backend, request):
    m = MtpModel(backend, LAYERS, VOCAB, seed=3, attention=KINDS[request.param])
    m.emb_host = m.embed_q4_0().reshape(VOCAB, (H // 32) * 18)
    m.host = [dict(h, qkv64=f8_ref.values(*h["qkv"]), out64=f8_ref.values(*h["out"])) for h in m.attention.host]
    yield m
    m.free()


def embedding(model, tokens):
    return np.stack([np.concatenate([orc.dequantize_q4_0(b) for b in model.emb_host[t].reshape(H // 32, 18)]) for t in tokens]).astype(np.float32)


def near(got, want, tol):
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4], tol[bad][:4])


def bf16(bits):
    return f8_ref.from_bf16(bits).astype(np.float64)


def caches(model, cache):
    """A traced cache's keys and values in 64 bits."""
    if model.attention.caches[0].type == "bf16":
        return [bf16(c) for c in cache]
    return [f8_ref.TABLE[c] * s[..., None].astype(np.float64) for c, s in zip(cache[:2], cache[2:])]


def check_attention(model, tr, host):
    att = model.attention
    nq, nk, d = att.heads
    at, t = tr["at"], tr["x"].shape[0]
    pos = at + np.arange(t)
    assert rel_err(tr["xn"], np.stack([orc.qwen_rmsnorm(r, host["norm"]) for r in tr["x"]])) < 1e-5
    want, tol = f8_ref.matmul(tr["xn"], host["qkv64"], True)
    rows = bf16(tr["rows"])
    near(rows, want, tol + (np.abs(want) + tol) * ref.BF16)
    per = att.q_width // d
    heads = rows[:, :nq * att.q_width].reshape(t, nq, per, d)
    gate = heads[:, :, 1] if att.gated else None
    k, v = rows[:, nq * att.q_width:].reshape(t, 2, nk, d).transpose(1, 0, 2, 3)
    want, tol = ref.heads_after(heads[:, :, 0], host["q_norm"], 1e-6, pos, att.frequencies, "half")
    q = bf16(tr["q"])
    near(q, want, tol + (np.abs(want) + tol) * ref.BF16)
    # the rows' keys and values, in the slots of their positions
    want_k, tol_k = ref.heads_after(k, host["k_norm"], 1e-6, pos, att.frequencies, "half")
    ck, cv = caches(model, tr["cache"])
    table = att.table
    for got, want, tol in ((ck, want_k, tol_k), (cv, v, np.zeros(v.shape))):
        got = ref.gathered(got, table, at + t)[at:]
        if att.caches[0].type == "bf16":
            near(got, want, tol + (np.abs(want) + tol) * ref.BF16)
        else:  # a step of e4m3, or of its smallest numbers, where the largest magnitude is 448; its f32 scale
            top = np.abs(want).max(2, keepdims=True) + tol
            near(got, want, tol + np.abs(want) * (2.0 ** -4 + 2.0 ** -21) + top / 448 * 2.0 ** -10)
    last = at + np.arange(t)
    keys, values = (bf16(tr["k"]), v) if tr["prompt"] else (ref.gathered(ck, table, at + t), ref.gathered(cv, table, at + t))
    want, tol = ref.attention(q, keys, values, last, d ** -0.5, gate)
    y = bf16(tr["y"])
    near(y, want, tol)
    want, tol = f8_ref.matmul(y.reshape(t, nq * d).astype(np.float32), host["out64"], True)
    near(tr["o"].astype(np.float64), want, tol + np.abs(want) * ref.F32)
    assert np.array_equal(tr["out"], tr["x"] + tr["o"])


def check_pass(model, tr, tokens, at, before):
    """A target pass over `tokens` at positions at..; `before`: each layer's cache before it, which it replaces."""
    trs = tr["attention"]
    assert [(a["layer"], a["at"], a["x"].shape[0]) for a in trs] == [(l, at, len(tokens)) for l in range(LAYERS)]
    x = embedding(model, tokens)
    for l, a in enumerate(trs):
        assert np.array_equal(a["x"], x) if l == 0 else rel_err(a["x"], x) < 1e-3
        check_attention(model, a, model.host[l])
        if before[l] is not None:  # what stood in front of the rows is as it was
            for new, old in zip(a["cache"], before[l]):
                new, old = [c if c.ndim == 4 else c[..., None] for c in (new, old)]
                assert np.array_equal(ref.gathered(new, model.attention.table, at), ref.gathered(old, model.attention.table, at))
        before[l] = a["cache"]
        x, _, _ = oracle_replay(model.parts[l], a["out"])
    n = tr["h"].shape[0]
    assert rel_err(tr["h"], x[-n:]) < 1e-3
    assert rel_err(tr["hn"], np.stack([orc.qwen_rmsnorm(r, model.norm_host) for r in tr["h"]])) < 1e-5
    for i in range(n):
        assert np.array_equal(tr["target"][i], orc.q6_k_matvec(model.lm_head_host, VOCAB, H, tr["hn"][i]))


def prompt_of(n):
    return [int(t) for t in np.random.default_rng(n).integers(0, VOCAB, n)]


@pytest.mark.parametrize("self_draft", [False, True], ids=["mtp_head", "self_draft"])
@pytest.mark.parametrize("n", [1, 8, 37])
def test_every_stage_of_every_pass(backend, model, self_draft, n):
    """Prompts over the cache (1, 8) and of their own rows (37); drafts that are mostly rejected, and mostly accepted."""
    eng = DeviceEngine(backend, model, k=K, temperature=T, greedy=True, seed=5, trace=True, self_draft=self_draft)
    loop = MtpLoop(eng, k=K, window=3)
    prompt = prompt_of(n)
    try:
        recs = loop.run(prompt, 5)
        length = eng.length
    finally:
        eng.free()
    before, at, boundary = [None] * LAYERS, 0, None
    for i, r in enumerate(recs):
        tokens = prompt if i == 0 else [boundary] + (r.trace["drafts"] if r.speculative else [])
        check_pass(model, r.trace, tokens, at, before)
        at += len(prompt) if i == 0 else r.accepted + 1 if r.speculative else 1
        boundary = r.emitted[-1]
    assert at == length == n + sum(len(r.emitted) for r in recs) - 1
    if self_draft:
        assert max(r.accepted for r in recs) > 0


def test_sequences_begin_anew(backend, model):
    """A second sequence on the engine gives what it gives alone: the first one's rows are not seen."""
    eng = DeviceEngine(backend, model, k=K, greedy=True, self_draft=True)
    try:
        loop = MtpLoop(eng, k=K)
        alone = [r.emitted for r in loop.run(prompt_of(12), 4)]
        MtpLoop(eng, k=K).run(prompt_of(61), 5)
        assert [r.emitted for r in MtpLoop(eng, k=K).run(prompt_of(12), 4)] == alone
    finally:
        eng.free()


def test_refusals(backend, model):
    eng = DeviceEngine(backend, model, k=K, greedy=True)
    most = model.attention.max_tokens
    try:
        for bad in ([], [VOCAB], [-1, 3], prompt_of(most + 1)):
            with pytest.raises(ValueError):
                eng.start(bad)
        t, _ = eng.start(prompt_of(most - 2))
        with pytest.raises(ValueError):
            eng.speculative(0, t)
        for step in range(2):
            t, _ = eng.plain(step, t)
        with pytest.raises(ValueError):
            eng.plain(2, t)
        with pytest.raises(ValueError):
            model.attention.forward(0, eng.d_h, 9, 1)
    finally:
        eng.free()


def test_one_sequence_at_a_time(backend, model):
    """Two engines on a model's caches: the one whose sequence was overwritten does not go on with the other's."""
    a, b = (DeviceEngine(backend, model, k=K, greedy=True) for _ in range(2))
    try:
        with pytest.raises(RuntimeError):
            a.plain(0, 5)
        t, _ = a.start(prompt_of(9))
        t, _ = a.plain(0, t)
        u, _ = b.start(prompt_of(10))
        for call in (a.plain, a.speculative):
            with pytest.raises(RuntimeError):
                call(1, t)
        b.speculative(0, u)
        a.start(prompt_of(9))
    finally:
        a.free(), b.free()
