"""Attention for prompts and for verify rows, and what goes before it, with their inputs.

Three operators around one cache, through the public entry points:

  rope     ``qk_rope_device``: an RMSNorm of every query and key head, the
           position rotation, and the new keys and values put into a paged cache;
  prompt   ``attn_prompt_device``: causal attention of packed prompts (or their
           last chunks: keys may reach back behind the queries), grouped heads;
  paged    ``attn_paged_device``: one or a few rows of every sequence (a token,
           or the verify rows of its drafts) over its pages of the cache, in bf16
           or in e4m3 with a scale for each token and head.

Both attentions may multiply their output by sigmoid(gate).  Plain forms compute
in 32 bits (the angles in 64: far positions need them) and round once.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
THETA, EPS = 1e7, 1e-6


# ---- the cases -----------------------------------------------------------------------
def listed():
    wide, usual = dict(q_heads=16, kv_heads=2, dim=256), dict(q_heads=32, kv_heads=8, dim=128)
    return [
        # one decode token's heads: latency alone
        dict(name="rope_t1", kind="rope", t=1, **wide, rotary=64, pairs="half", x="f32", packed=False, page=16),
        # rows of several prompts, the other order of pairs, 32-bit projections
        dict(name="rope_t515", kind="rope", t=515, **usual, rotary=128, pairs="neighbours", x="f32", packed=True, page=64),
        # the largest prompt chunk
        dict(name="rope_t4096", kind="rope", t=4096, **wide, rotary=64, pairs="half", x="bf16", packed=True, page=64),
        # a short prompt
        dict(name="prompt_37", kind="prompt", seqs=1, low=37, high=37, context=0, **wide, gate=True),
        # a batch of short and middling prompts, some with their first part in place already
        dict(name="prompt_packed", kind="prompt", seqs=24, low=1, high=700, context=300, **usual, gate=False),
        # the largest chunk of one prompt, gated heads
        dict(name="prompt_4096", kind="prompt", seqs=1, low=4096, high=4096, context=0, **wide, gate=True),
        # a long prompt in one piece
        dict(name="prompt_8192", kind="prompt", seqs=1, low=8192, high=8192, context=0, **usual, gate=False),
        # one user's next token: latency
        dict(name="paged_1x1000", kind="paged", seqs=1, rows=1, low=1000, high=1000, **wide, page=16, cache="bf16", gate=True),
        # the same far into a long document
        dict(name="paged_1x131072", kind="paged", seqs=1, rows=1, low=131072, high=131072, **wide, page=64, cache="bf16", gate=True),
        # verify rows of three drafts in a busy server, lengths of all sizes
        dict(name="paged_64_verify", kind="paged", seqs=64, rows=4, low=50, high=8192, **wide, page=16, cache="bf16", gate=True),
        # tokens of a busy server over an 8-bit cache
        dict(name="paged_96_f8", kind="paged", seqs=96, rows=1, low=50, high=8192, **usual, page=32, cache="f8", gate=False),
        # the largest batch
        dict(name="paged_256", kind="paged", seqs=256, rows=1, low=3500, high=4500, **usual, page=64, cache="bf16", gate=False),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["rope", "prompt", "prompt", "paged", "paged"])
    dim, kv = rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 4, 8])
    heads = dict(q_heads=kv * rng.choice([1, 2, 3, 4, 7, 8] if kv < 8 else [1, 2, 4]), kv_heads=kv, dim=dim)
    page = rng.choice([16, 32, 64, 128])
    if kind == "rope":
        return dict(kind=kind, t=_log_int(rng, 1, 4096), **heads, rotary=rng.choice([0, 32, dim // 2, dim]), pairs=rng.choice(["half", "neighbours"]),
                    x=rng.choice(["f32", "bf16"]), packed=rng.random() < 0.5, page=page)
    if kind == "prompt":
        seqs, high = _log_int(rng, 1, 32), _log_int(rng, 4, 8192)
        high = min(high, int(math.sqrt(32 * 8192.0 ** 2 / (seqs * heads["q_heads"]))))
        return dict(kind=kind, seqs=seqs, low=max(1, int(high * rng.random())), high=high, context=rng.choice([0, 0, high // 4]), **heads,
                    gate=rng.random() < 0.5)
    seqs, high = _log_int(rng, 1, 256), _log_int(rng, 16, 131072)
    high = max(16, min(high, int(256 * 3500 * 8 * 128 / (seqs * kv * dim))))
    return dict(kind=kind, seqs=seqs, rows=rng.choice([1, 1, 2, 4, 8]), low=max(8, int(high * rng.random())), high=high, **heads, page=page,
                cache=rng.choice(["bf16", "f8"]), gate=rng.random() < 0.5)


def _lengths(c):
    """The sequences' lengths: spread over low..high (evenly over their logarithm), in an order that is not theirs; the longest
    is `high`.  They belong to the case, as its sizes do."""
    n = c["seqs"]
    g = torch.Generator().manual_seed(n * 31 + c["high"])
    at = torch.rand(n, generator=g, dtype=torch.float64)
    at[n // 2] = 1.0
    span = math.log(c["high"] / c["low"])
    return [min(c["high"], max(c["low"], int(round(c["low"] * math.exp(span * v))))) for v in at.tolist()]


def _contexts(c):
    """How many keys of each prompt lie before its queries: none, or up to `context` for about half of them."""
    g = torch.Generator().manual_seed(c["seqs"] * 17 + c["high"])
    some = torch.rand(c["seqs"], 2, generator=g, dtype=torch.float64).tolist()
    return [int(a * c["context"]) if b < 0.5 else 0 for a, b in some]


# ---- inputs --------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _normal(shape, seed, std=1.0):
    return torch.randn(shape, generator=_gen(seed), device=DEV) * std


def _keys(shape, seed, dim):
    """Keys after their norm and rotation: N(0, 1) and a part that all have in common, as trained heads have it."""
    return _normal(shape, seed) + 0.7 * _normal((dim,), seed + 1)


def _bf16(x):
    return x.to(torch.bfloat16).contiguous()


def _steps(*lengths):
    return torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32, device=DEV)


_BACKEND = []


def _backend():
    if not _BACKEND:
        from turboqwenfare_amd.backend import HipBackend
        _BACKEND.append(HipBackend())
    return _BACKEND[0]


def _buf(t):
    """A device buffer from a tensor's first element to the end of its storage."""
    from turboqwenfare_amd.backend import DeviceBuffer
    return DeviceBuffer(t.data_ptr(), t.untyped_storage().nbytes() - t.storage_offset() * t.element_size())


class _Kept:
    """Handles of the framework, given back with the state."""

    def __init__(self, handles, free):
        self.handles, self.free = handles, free

    def __del__(self):
        for h, f in zip(self.handles, self.free):
            f(h)


def _frequencies(rotary):
    return [THETA ** (-2.0 * i / rotary) for i in range(rotary // 2)]


def _prepare_rope(c, s):
    t, hq, hk, d = c["t"], c["q_heads"], c["kv_heads"], c["dim"]
    kind = torch.float32 if c["x"] == "f32" else torch.bfloat16
    # what a projection of all heads gives: a token's query heads, then its key and value heads
    rows = (_normal((t, hq + 2 * hk, d), s) * 1.5).to(kind)
    pages = -(-t // c["page"]) + 3
    first = int(torch.randint(0, 200000, (1,), generator=torch.Generator().manual_seed(s)))
    order = torch.randperm(pages, generator=_gen(s + 5), device=DEV)
    token = torch.arange(t, device=DEV)
    shape = (pages, hk, c["page"], d)
    return dict(q=rows[:, :hq], k=rows[:, hq:hq + hk], v=rows[:, hq + hk:], wq=1.0 + 0.1 * _normal((d,), s + 1), wk=1.0 + 0.1 * _normal((d,), s + 2),
                positions=(first + token).int(), slots=(order[token // c["page"]] * c["page"] + token % c["page"]).int(),
                freq=torch.tensor(_frequencies(c["rotary"]), dtype=torch.float64, device=DEV),
                q_out=torch.zeros(t, hq, d, dtype=torch.bfloat16, device=DEV),
                k_out=torch.zeros(t, hk, d, dtype=torch.bfloat16, device=DEV) if c["packed"] else None,
                k_cache=torch.zeros(shape, dtype=torch.bfloat16, device=DEV), v_cache=torch.zeros(shape, dtype=torch.bfloat16, device=DEV),
                status=torch.zeros(1, dtype=torch.int32, device=DEV))


def _prepare_prompt(c, s):
    hq, hk, d = c["q_heads"], c["kv_heads"], c["dim"]
    lq, ctx = _lengths(c), _contexts(c)
    lk = [a + b for a, b in zip(lq, ctx)]
    tq, tk = sum(lq), sum(lk)
    # queries and keys as the rotation left them; values (and gates) where the projections put them, among other heads
    return dict(q=_bf16(_normal((tq, hq, d), s)), k=_bf16(_keys((tk, hk, d), s + 1, d)), v=_bf16(_normal((tk, 2 * hk, d), s + 3))[:, hk:],
                gate=_bf16(_normal((tq, hq, 2 * d), s + 4))[:, :, d:] if c["gate"] else None, cu_q=_steps(*lq), cu_k=_steps(*lk),
                lq=lq, lk=lk, y=torch.zeros(tq, hq, d, dtype=torch.bfloat16, device=DEV), status=torch.zeros(1, dtype=torch.int32, device=DEV))


def _f8(x):
    """(values, scales) of rows [..., d]: the largest magnitude of each becomes 448."""
    scale = x.abs().amax(-1) / 448.0
    return (x / scale.unsqueeze(-1)).to(torch.float8_e4m3fn), scale


def _prepare_paged(c, s):
    n, hq, hk, d, page = c["seqs"], c["q_heads"], c["kv_heads"], c["dim"], c["page"]
    lens = _lengths(c)
    need = [-(-v // page) for v in lens]
    pages = sum(need) + 1
    ids = torch.randperm(pages, generator=_gen(s + 5), device=DEV).int()
    width = max(need)
    table = torch.full((n, width), -1, dtype=torch.int32, device=DEV)
    at = torch.tensor([0, *need], device=DEV).cumsum(0)[:-1]
    col = torch.arange(width, device=DEV)
    used = col[None, :] < torch.tensor(need, device=DEV)[:, None]
    table[used] = ids[(at[:, None] + col)[used]]
    shape = (pages, hk, page, d)
    k, v = _keys(shape, s + 1, d), _normal(shape, s + 3)
    if c["cache"] == "f8":
        (k, ks), (v, vs) = _f8(k), _f8(v)
    else:
        k, ks, v, vs = _bf16(k), None, _bf16(v), None
    t = n * c["rows"]
    return dict(q=_bf16(_normal((t, hq, d), s)), k=k, v=v, ks=ks, vs=vs, table=table, lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
                gate=_bf16(_normal((t, hq, 2 * d), s + 4))[:, :, d:] if c["gate"] else None,
                y=torch.zeros(t, hq, d, dtype=torch.bfloat16, device=DEV), status=torch.zeros(1, dtype=torch.int32, device=DEV))


def prepare(case, seed):
    c, s = dict(case), 1_000_003 * int(seed) + 17
    st = {"rope": _prepare_rope, "prompt": _prepare_prompt, "paged": _prepare_paged}[c["kind"]](c, s)
    st["c"] = c
    torch.cuda.synchronize()
    if own:
        be = st["be"] = _backend()
        st["b"] = {k: _buf(v) for k, v in st.items() if isinstance(v, torch.Tensor)}
        b = st["b"]
        if c["kind"] == "rope":
            wq, wk = be.upload_f32(st["wq"].cpu().numpy()), be.upload_f32(st["wk"].cpu().numpy())
            rope = be.prepare_rope(_frequencies(c["rotary"])) if c["rotary"] else None
            st["kept"] = _Kept([wq, wk] + [rope] * bool(rope), [be.free_tensor, be.free_tensor, be.free_rope])
            st["wq"], st["wk"], st["rope"] = wq, wk, rope
            st["cache"] = be.kv_cache(b["k_cache"], b["v_cache"], *st["k_cache"].shape)
        if c["kind"] == "paged":
            st["cache"] = be.kv_cache(b["k"], b["v"], *st["k"].shape, type=c["cache"], d_k_scales=b.get("ks"), d_v_scales=b.get("vs"))
    return st


# ---- plain forms ---------------------------------------------------------------------------
def _normed(x, w):
    x = x.float()
    return x * (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)) * w


def _rotated(x, angle, pairs):
    """x [t, heads, d] turned by angle [t, rotary / 2]; what is past the rotary part stays."""
    n = angle.shape[1]
    if n == 0:
        return x
    part, rest = x[..., :2 * n], x[..., 2 * n:]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    if pairs == "half":
        a, b = part[..., :n], part[..., n:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
    a, b = part[..., 0::2], part[..., 1::2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)


def _gated(y, gate):
    return y if gate is None else y / (1.0 + torch.exp(-gate.float()))


def _softmax_rows(s, seen):
    """Weights of the scores that are seen; rows that see nothing are zero."""
    s = torch.where(seen, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, 1.0)


def _attend(q, k, v, seen):
    """q [n, rows, q_heads, d], k and v [n, keys, kv_heads, d] f32, seen [n, rows, keys] -> [n, rows, q_heads, d]."""
    n, r, hq, d = q.shape
    hk, g = k.shape[2], hq // k.shape[2]
    qs = q.view(n, r, hk, g, d).permute(0, 2, 1, 3, 4).reshape(n * hk, r * g, d)
    ks = k.permute(0, 2, 3, 1).reshape(n * hk, d, -1)
    vs = v.permute(0, 2, 1, 3).reshape(n * hk, -1, d)
    s = torch.bmm(qs, ks) * d ** -0.5
    p = _softmax_rows(s.view(n, hk, r, g, -1), seen[:, None, :, None, :])
    y = torch.bmm(p.view(n * hk, r * g, -1), vs)
    return y.view(n, hk, r, g, d).permute(0, 2, 1, 3, 4).reshape(n, r, hq, d)


def _plain_rope(st):
    c = st["c"]
    angle = st["positions"].double()[:, None] * st["freq"]
    q = _rotated(_normed(st["q"], st["wq"]), angle, c["pairs"]).to(torch.bfloat16)
    k = _rotated(_normed(st["k"], st["wk"]), angle, c["pairs"]).to(torch.bfloat16)
    v = st["v"].to(torch.bfloat16)
    page, slot = st["slots"].long() // c["page"], st["slots"].long() % c["page"]
    st["k_cache"][page, :, slot] = k
    st["v_cache"][page, :, slot] = v
    return dict(q=q, k=k if c["packed"] else None, k_cache=st["k_cache"], v_cache=st["v_cache"])


def _plain_prompt(st):
    """Sequences side by side, padded to the longest."""
    lq, lk = st["cu_q"].diff(), st["cu_k"].diff()
    row, col = torch.arange(max(st["lq"]), device=DEV), torch.arange(max(st["lk"]), device=DEV)
    real, key = row < lq[:, None], col < lk[:, None]
    at_q = torch.where(real, st["cu_q"][:-1, None] + row, 0).long()
    at_k = torch.where(key, st["cu_k"][:-1, None] + col, 0).long()
    seen = key[:, None, :] & (col <= row[:, None] + (lk - lq)[:, None, None])
    y = _attend(st["q"].float()[at_q], st["k"].float()[at_k], st["v"].float()[at_k], seen)
    return _gated(y[real], st["gate"]).to(torch.bfloat16)


def _plain_paged(st):
    c = st["c"]
    n, page = c["seqs"], c["page"]
    table = st["table"].clamp(min=0).long()

    def rows(x, scale):
        x = (x.view(torch.uint8)[table].view(x.dtype).float() * scale[table].unsqueeze(-1)) if scale is not None else x[table].float()
        return x.transpose(2, 3).reshape(n, -1, c["kv_heads"], c["dim"])  # [n, pages, heads, slots, d] -> [n, keys, heads, d]

    col, row = torch.arange(table.shape[1] * page, device=DEV), torch.arange(c["rows"], device=DEV)
    seen = col <= (st["lens"][:, None] - c["rows"] + row)[:, :, None]
    y = _attend(st["q"].float().view(n, c["rows"], c["q_heads"], c["dim"]), rows(st["k"], st["ks"]), rows(st["v"], st["vs"]), seen)
    return _gated(y.flatten(0, 1), st["gate"]).to(torch.bfloat16)


# ---- one pass ---------------------------------------------------------------------------------
def run(st):
    c, kind = st["c"], st["c"]["kind"]
    if not own:
        return {"rope": _plain_rope, "prompt": _plain_prompt, "paged": _plain_paged}[kind](st)
    be, b, heads = st["be"], st["b"], (c["q_heads"], c["kv_heads"], c["dim"])
    strides = lambda t: (t.stride(0), t.stride(1))  # noqa: E731
    gate = dict(d_gate=b["gate"], gate_strides=strides(st["gate"])) if c.get("gate") else {}
    if kind == "rope":
        be.qk_rope_device(b["q"], b["k"], b["v"], c["t"], heads, b["positions"], b["q_out"], d_k_out=b.get("k_out"), x_type=c["x"],
                          strides=(strides(st["q"]), strides(st["k"]), strides(st["v"])), q_norm=st["wq"], k_norm=st["wk"], eps=EPS,
                          rope=st["rope"], pairs=c["pairs"], cache=st["cache"], d_slots=b["slots"], d_status=b["status"])
        return dict(q=st["q_out"], k=st["k_out"], k_cache=st["k_cache"], v_cache=st["v_cache"])
    if kind == "prompt":
        be.attn_prompt_device(b["q"], b["k"], b["v"], heads, b["cu_q"], b["cu_k"], c["seqs"], st["q"].shape[0], st["k"].shape[0], b["y"],
                              strides=(strides(st["q"]), strides(st["k"]), strides(st["v"])), d_status=b["status"], **gate)
        return st["y"]
    be.attn_paged_device(b["q"], heads, c["seqs"], c["rows"], st["cache"], b["table"], st["table"].shape[1], b["lens"], b["y"],
                         d_status=b["status"], **gate)
    return st["y"]


# ---- the same from the definitions, in 64 bits ---------------------------------------------
def _exact_head(q, k, v, last):
    """One query head: q [rows, d], k and v [keys, d], last [rows]: the last key that each row sees (-1: none)."""
    s = q @ k.T / math.sqrt(q.shape[1])
    s.masked_fill_(torch.arange(k.shape[0], device=DEV) > last[:, None], -math.inf)
    return torch.softmax(s, 1).nan_to_num_(0.0) @ v


def _exact_sequence(out, q, k, v, gate, last):
    group = q.shape[1] // k.shape[1]
    for h in range(q.shape[1]):
        y = _exact_head(q[:, h].double(), k[:, h // group], v[:, h // group], last)
        out[:, h] = y if gate is None else y * torch.sigmoid(gate[:, h].double())


def _exact_rope(st):
    c = st["c"]
    n, d = c["rotary"] // 2, c["dim"]
    a = st["positions"].double()[:, None] * st["freq"]
    turn = torch.eye(d, dtype=torch.float64, device=DEV).repeat(c["t"], 1, 1)  # each token's rotation as a matrix
    for i in range(n):
        x, y = (i, i + n) if c["pairs"] == "half" else (2 * i, 2 * i + 1)
        turn[:, x, x] = turn[:, y, y] = a[:, i].cos()
        turn[:, x, y] = -a[:, i].sin()
        turn[:, y, x] = a[:, i].sin()
    out = {}
    for name, w in (("q", st["wq"]), ("k", st["wk"])):
        x = st[name].double()
        x = x * torch.rsqrt(x.square().mean(2, keepdim=True) + EPS) * w.double()
        out[name] = torch.bmm(x, turn.transpose(1, 2).contiguous())
    caches = [torch.zeros(st["k_cache"].shape, dtype=torch.float64, device=DEV) for _ in range(2)]
    flat = st["slots"].long()
    for cache, x in zip(caches, (out["k"], st["v"].double())):
        by_slot = cache.transpose(1, 2).reshape(-1, c["kv_heads"], d)  # a copy: [slots, heads, d]
        by_slot[flat] = x
        cache.copy_(by_slot.view(cache.shape[0], c["page"], c["kv_heads"], d).transpose(1, 2))
    return dict(q=out["q"], k=out["k"] if c["packed"] else None, k_cache=caches[0], v_cache=caches[1])


def _e4m3_table():
    """The 256 values of e4m3: sign, 4 exponent bits (bias 7), 3 fraction bits; 0x7F is not a number."""
    b = torch.arange(256, device=DEV)
    ex, fr = ((b >> 3) & 15).double(), (b & 7).double()
    v = torch.where(ex == 0, fr / 8 * 2.0 ** -6, (1 + fr / 8) * torch.exp2(ex - 7))
    v = torch.where((b & 127) == 127, math.nan, v)
    return torch.where(b >= 128, -v, v)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    c = st["c"]
    if c["kind"] == "rope":
        return _exact_rope(st)
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    gate = lambda a, b: st["gate"][a:b] if c["gate"] else None  # noqa: E731
    if c["kind"] == "prompt":
        q0 = k0 = 0
        for lq, lk in zip(st["lq"], st["lk"]):
            last = torch.arange(lq, device=DEV) + (lk - lq)
            _exact_sequence(out[q0:q0 + lq], st["q"][q0:q0 + lq], st["k"][k0:k0 + lk].double(), st["v"][k0:k0 + lk].double(), gate(q0, q0 + lq), last)
            q0, k0 = q0 + lq, k0 + lk
        return out
    r, values = c["rows"], _e4m3_table()
    for i, n in enumerate(st["lens"].tolist()):
        ids = st["table"][i, :-(-n // c["page"])].long()

        def flat(x, s):
            if s is not None:
                x = values[x.view(torch.uint8)[ids].long()] * s[ids].double().unsqueeze(-1)
            else:
                x = x[ids].double()
            return x.transpose(1, 2).flatten(0, 1)[:n]

        last = torch.arange(n - r, n, device=DEV)
        a = i * r
        _exact_sequence(out[a:a + r], st["q"][a:a + r], flat(st["k"], st["ks"]), flat(st["v"], st["vs"]), gate(a, a + r), last)
    return out


# ---- what a pass cannot do without ------------------------------------------------------------
def work(case):
    c = case
    hq, hk, d = c["q_heads"], c["kv_heads"], c["dim"]
    if c["kind"] == "rope":  # a value counts as 8 operations: its norm, its weight, its turn
        size = 4 if c["x"] == "f32" else 2
        return dict(bytes=c["t"] * d * ((hq + 2 * hk) * (size + 2) + (2 * hk if c["packed"] else 0)), flops=8.0 * c["t"] * d * (hq + hk))
    lens = _lengths(c)
    if c["kind"] == "prompt":
        lk = [a + b for a, b in zip(lens, _contexts(c))]
        seen = sum(n * (k - n) + n * (n + 1) / 2 for n, k in zip(lens, lk))
        return dict(bytes=2 * d * (sum(lens) * hq * (3 if c["gate"] else 2) + 2 * sum(lk) * hk), flops=4.0 * d * hq * seen)
    r, size = c["rows"], 1 if c["cache"] == "f8" else 2
    keys = 2.0 * sum(lens) * hk * (d * size + (4 if c["cache"] == "f8" else 0))
    return dict(bytes=keys + 2.0 * c["seqs"] * r * hq * d * (3 if c["gate"] else 2), flops=4.0 * d * hq * r * sum(lens))
