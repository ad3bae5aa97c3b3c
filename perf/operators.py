"""The batched router and the 8-bit floating point products, with their inputs.

Four operators that a server runs over the rows of a batch (the verify rows of
many sequences, or a chunk of a prompt), through the public entry points:

  logits   the router's product ``router_logits_device``: x [t, hidden] times
           the f32 router [experts, hidden];
  route    ``route_tokens_device``: scores (softmax or sigmoid), a bias for
           choosing only, groups, top-k with ties to the lowest index,
           renormalised weights;
  matmul   ``f8_matmul_device``: rows quantised to e4m3 in blocks of 128 times
           an e4m3 matrix with a scale for each block of 128 x 128;
  experts  ``f8_experts_device``: the routed experts' gate, up (SwiGLU) and
           down products in the same format, and their weighted sum.

An e4m3 row block of 128 values has the scale a / 448 (a: its largest
magnitude) and the values x * (448 / a) rounded to nearest even; a block whose
largest magnitude is below 2^-100 is zero.  Plain forms take the quantised
values as they are and compute in 32 bits; routing is in 64, since ids have to
be equal and scores next to each other are not rare.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

H, F, E, TOP_K, V = 2048, 512, 256, 8, 151936
DEV = "cuda"
NONE = -1  # the id of an empty slot, 0xFFFF as int16
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ---- the cases -----------------------------------------------------------------------
def listed():
    return [
        # one decode token's router product and routes: latency alone
        dict(name="logits_t1", kind="logits", t=1, hidden=H, experts=E, x="f32"),
        dict(name="route_t1", kind="route", t=1, experts=E, top_k=TOP_K, score="softmax", groups=1, top_groups=1, best=1,
             renorm=True, scale=1.0, bias=False, masked=0.0, logits="f32"),
        # the same for the largest prompt chunk: a router balanced by a bias over groups, some rows padding
        dict(name="logits_t4096", kind="logits", t=4096, hidden=H, experts=E, x="bf16"),
        dict(name="route_t4096", kind="route", t=4096, experts=E, top_k=TOP_K, score="sigmoid", groups=8, top_groups=4, best=2,
             renorm=True, scale=2.5, bias=True, masked=0.02, logits="f32"),
        # one expert-sized matrix against one token
        dict(name="matmul_t1", kind="matmul", t=1, rows=F, cols=H, x="f32", y="f32"),
        # the LM head over the verify rows of two sequences
        dict(name="matmul_head_t8", kind="matmul", t=8, rows=V, cols=H, x="bf16", y="f32"),
        # sizes that fit no tile, a prompt's tail
        dict(name="matmul_t37_odd", kind="matmul", t=37, rows=1000, cols=1100, x="f32", y="bf16"),
        # a projection over the largest prompt chunk
        dict(name="matmul_t4096", kind="matmul", t=4096, rows=8192, cols=4096, x="bf16", y="bf16"),
        # one decode token through the experts of four layers (so that their weights are not in a cache already)
        dict(name="experts_t1", kind="experts", t=1, hidden=H, width=F, experts=E, top_k=TOP_K, skew=1.1, empty=0.0, layers=4, x="bf16"),
        # a prompt's tail, or the verify rows of nine sequences, some rows padding
        dict(name="experts_t37", kind="experts", t=37, hidden=H, width=F, experts=E, top_k=TOP_K, skew=1.1, empty=0.05, layers=1, x="bf16"),
        # an ordinary chunk with the skewed expert popularity of real routers
        dict(name="experts_t512", kind="experts", t=512, hidden=H, width=F, experts=E, top_k=TOP_K, skew=1.1, empty=0.0, layers=1, x="bf16"),
        # the largest chunk, experts evenly used
        dict(name="experts_t4096", kind="experts", t=4096, hidden=H, width=F, experts=E, top_k=TOP_K, skew=0.0, empty=0.0, layers=1, x="bf16"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["logits", "route", "route", "matmul", "matmul", "experts", "experts"])
    x = rng.choice(["f32", "bf16"])
    if kind == "logits":
        return dict(kind=kind, t=_log_int(rng, 1, 4096), hidden=_log_int(rng, 64, H), experts=_log_int(rng, 8, 256), x=x)
    if kind == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        per = max(2, _log_int(rng, 16, 512) // groups)
        kept = rng.randint(1, groups)
        return dict(kind=kind, t=_log_int(rng, 1, 4096), experts=groups * per, top_k=rng.randint(1, min(16, kept * per)),
                    score=rng.choice(["softmax", "sigmoid"]), groups=groups, top_groups=kept, best=rng.choice([1, 2]),
                    renorm=rng.random() < 0.7, scale=rng.choice([1.0, 2.5]), bias=rng.random() < 0.5,
                    masked=rng.choice([0.0, 0.05]), logits=x)
    if kind == "matmul":
        t, rows = _log_int(rng, 1, 4096), _log_int(rng, 16, 16384)
        cols = min(_log_int(rng, 64, 8192), int(4096 * 8192 * 4096 / (t * rows)))
        return dict(kind=kind, t=t, rows=rows, cols=cols, x=x, y=rng.choice(["f32", "bf16"]))
    experts = rng.choice([8, 60, 128, 256])
    return dict(kind=kind, t=_log_int(rng, 1, 4096), hidden=rng.choice([1024, 2048, rng.randint(200, 2048)]),
                width=rng.choice([256, 512, rng.randint(64, 512)]), experts=experts, top_k=rng.randint(1, 8),
                skew=rng.choice([0.0, 0.7, 1.1]), empty=rng.choice([0.0, 0.1]), layers=1, x=x)


# ---- inputs --------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _normal(shape, seed, std=1.0):
    return torch.randn(shape, generator=_gen(seed), device=DEV) * std


def _rows(t, cols, kind, seed):
    """Hidden rows after a norm: N(0, 1) with a few channels that are much larger, as models have them."""
    channel = torch.where(torch.rand(cols, generator=_gen(9), device=DEV) < 0.01, 8.0, 1.0)
    return (_normal((t, cols), seed) * channel).to(TYPES[kind]).contiguous()


def _blocks(n):
    return -(-n // 128)


def _f8_weights(n, rows, cols, seed):
    """n matrices N(0, 1 / cols) as e4m3 [n, rows, cols] with f32 scales [n, rows / 128, cols / 128] (rounded up)."""
    br, bc = _blocks(rows), _blocks(cols)
    q = torch.empty(n, rows, cols, dtype=torch.float8_e4m3fn, device=DEV)
    s = torch.empty(n, br, bc, device=DEV)
    for at in range(0, n, 32):  # 32 matrices at a time: room for their 32-bit values
        k = min(32, n - at)
        w = torch.zeros(k, br * 128, bc * 128, device=DEV)
        w[:, :rows, :cols] = _normal((k, rows, cols), seed + 7919 * at, cols ** -0.5)
        a = w.view(k, br, 128, bc, 128).abs().amax((2, 4))
        s[at:at + k] = a / 448.0
        w = (w.view(k, br, 128, bc, 128) / s[at:at + k, :, None, :, None]).view_as(w)
        q[at:at + k] = w[:, :rows, :cols].to(torch.float8_e4m3fn)
    return q, s


_LAYERS = {}  # the experts' weights of the geometry in use, by layer


def _layer(c, index):
    """(gate, up, down) of a layer, each (values, scales): made once for a geometry, as a server keeps them."""
    key = (c["experts"], c["hidden"], c["width"])
    if _LAYERS and next(iter(_LAYERS))[0] != key:
        _LAYERS.clear()
    if (key, index) not in _LAYERS:
        n, hidden, width = key
        _LAYERS[key, index] = [_f8_weights(n, r, k, 1000 * index + 10 + i)
                               for i, (r, k) in enumerate(((width, hidden), (width, hidden), (hidden, width)))]
    return _LAYERS[key, index]


def _routes(t, experts, top_k, skew, empty, seed):
    """Routes of t tokens from a Zipf(skew) popularity; a share `empty` of the rows is padding."""
    rng = np.random.default_rng(seed)
    rank = rng.permutation(experts)
    scores = -skew * np.log(rank + 1.0)[None, :] + rng.gumbel(size=(t, experts))
    ids = np.argsort(-scores, axis=1, kind="stable")[:, :top_k]
    p = np.exp(np.take_along_axis(scores, ids, 1) - scores.max(1, keepdims=True))
    p = p / p.sum(1, keepdims=True)
    pad = rng.random(t) < empty
    ids[pad], p[pad] = NONE, 0.0
    return torch.from_numpy(ids.astype(np.int16)).to(DEV), torch.from_numpy(p.astype(np.float32)).to(DEV)


_BACKEND, _HANDLES = [], {}


def _backend():
    if not _BACKEND:
        from turboqwenfare_amd.backend import HipBackend
        _BACKEND.append(HipBackend())
    return _BACKEND[0]


def _buf(t):
    from turboqwenfare_amd.backend import DeviceBuffer
    return DeviceBuffer(t.data_ptr(), t.numel() * t.element_size())


class _Kept:
    """Handles of the framework, given back with the state."""

    def __init__(self, handles, free):
        self.handles, self.free = handles, free

    def __del__(self):
        for h in self.handles:
            self.free(h)


def _experts_handle(c, index):
    """The prepared experts of a layer, with their matrices: laid out once for a geometry, and given back when neither
    a state nor this module, which keeps those of the newest geometry, has them."""
    be, key = _backend(), (c["experts"], c["hidden"], c["width"], index)
    if _HANDLES and next(iter(_HANDLES))[:3] != key[:3]:
        _HANDLES.clear()
    if key not in _HANDLES:
        layer = _layer(c, index)
        torch.cuda.synchronize()
        mats = [[be.upload_f8_device(_buf(q[e]), _buf(s[e]), q.shape[1], q.shape[2]) for e in range(q.shape[0])]
                for q, s in layer]
        prepared = be.prepare_f8_experts(*mats)
        _HANDLES[key] = _Kept([prepared, *mats[0], *mats[1], *mats[2]],
                              lambda h: be.free_f8_experts(h) if h is prepared else be.free_weights(h))
    return _HANDLES[key]


def prepare(case, seed):
    c, s = dict(case), 1_000_003 * int(seed) + 17
    kind, t = c["kind"], c["t"]
    st = dict(c=c)
    if kind == "logits":
        st.update(x=_rows(t, c["hidden"], c["x"], s), w=_normal((c["experts"], c["hidden"]), s + 1, c["hidden"] ** -0.5),
                  out=torch.zeros(t, c["experts"], device=DEV))
    elif kind == "route":
        lg = _normal((t, c["experts"]), s, 1.5)
        if c["masked"]:  # experts that are out of service, and padding rows
            lg[torch.rand(lg.shape, generator=_gen(s + 1), device=DEV) < c["masked"]] = -math.inf
            lg[torch.rand(t, generator=_gen(s + 2), device=DEV) < c["masked"]] = -math.inf
        st.update(x=lg.to(TYPES[c["logits"]]).contiguous(), bias=_normal((c["experts"],), s + 3, 0.05) if c["bias"] else None,
                  ids=torch.zeros(t, c["top_k"], dtype=torch.int16, device=DEV), w=torch.zeros(t, c["top_k"], device=DEV),
                  status=torch.zeros(1, dtype=torch.int32, device=DEV))
    elif kind == "matmul":
        q, sc = _f8_weights(1, c["rows"], c["cols"], s + 1)
        st.update(x=_rows(t, c["cols"], c["x"], s), q=q[0], s=sc[0], out=torch.zeros(t, c["rows"], dtype=TYPES[c["y"]], device=DEV))
    else:
        routes = [_routes(t, c["experts"], c["top_k"], c["skew"], c["empty"], (s, i)) for i in range(c["layers"])]
        st.update(x=[_rows(t, c["hidden"], c["x"], s + 10 * i) for i in range(c["layers"])], ids=[r[0] for r in routes], w=[r[1] for r in routes],
                  out=[torch.zeros(t, c["hidden"], dtype=torch.bfloat16, device=DEV) for _ in range(c["layers"])],
                  status=torch.zeros(1, dtype=torch.int32, device=DEV), layers=[_layer(c, i) for i in range(c["layers"])])
    if own:
        torch.cuda.synchronize()
        be = st["be"] = _backend()
        if kind == "logits":
            w = be.upload_f32(st["w"].cpu().numpy())
            st["kept"] = _Kept([w], be.free_tensor)
        elif kind == "matmul":
            w = be.upload_f8_device(_buf(st["q"]), _buf(st["s"]), c["rows"], c["cols"])
            st["kept"] = _Kept([w], be.free_weights)
        elif kind == "experts":
            st["handles"] = [_experts_handle(c, i) for i in range(c["layers"])]
        st["b"] = {k: [_buf(u) for u in v] if isinstance(v, list) else _buf(v)
                   for k, v in st.items() if k in ("x", "bias", "ids", "w", "out", "status") and v is not None}
    torch.cuda.synchronize()
    return st


# ---- plain forms ---------------------------------------------------------------------------
def _quantised(x):
    """The values of the rows after quantisation to e4m3 in blocks of 128, f32."""
    t, n = x.shape
    p = torch.zeros(t, _blocks(n) * 128, device=x.device)
    p[:, :n] = x
    p = p.view(t, -1, 128)
    a = p.abs().amax(2, keepdim=True).double()
    zero = a < 2.0 ** -100
    s = torch.where(zero, 0.0, a / 448.0).float()
    inv = torch.where(zero, 0.0, 448.0 / a).float()
    return ((p * inv).to(torch.float8_e4m3fn).float() * s).view(t, -1)[:, :n]


def _values(q, s):
    """The f32 values of e4m3 matrices [..., rows, cols] with block scales."""
    rows, cols = q.shape[-2:]
    s = s.repeat_interleave(128, -2)[..., :rows, :].repeat_interleave(128, -1)[..., :cols]
    return q.float() * s


def _route(c, lg, bias):
    t, n = lg.shape
    lg = lg.double()
    bad = (lg.isnan() | (lg == math.inf)).any(1, keepdim=True)
    off = lg == -math.inf
    if c["score"] == "softmax":
        top = lg.amax(1, keepdim=True)
        e = torch.where(off, 0.0, torch.exp(lg - torch.where(top == -math.inf, 0.0, top)))
        score = e / torch.where(top == -math.inf, 1.0, e.sum(1, keepdim=True))
    else:
        score = 1.0 / (1.0 + torch.exp(-lg))
    choose = score + (bias.double() if bias is not None else 0.0)
    choose = torch.where(off | bad, -math.inf, choose)
    if c["groups"] > 1:
        per = choose.view(t, c["groups"], -1)
        best = per.topk(min(c["best"], per.shape[2]), 2).values
        group = torch.where(best[:, :, :1] == -math.inf, -math.inf, torch.where(best == -math.inf, 0.0, best).sum(2, keepdim=True))
        order = group.squeeze(2).sort(dim=1, descending=True, stable=True).indices[:, :c["top_groups"]]
        keep = torch.zeros(t, c["groups"], dtype=torch.bool, device=lg.device).scatter_(1, order, True)
        choose = torch.where(keep[:, :, None], per, -math.inf).view(t, n)
    value, ids = choose.sort(dim=1, descending=True, stable=True)
    value, ids = value[:, :c["top_k"]], ids[:, :c["top_k"]]
    none = value == -math.inf
    w = torch.where(none, 0.0, score.gather(1, ids))
    if c["renorm"]:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
    return torch.where(none, NONE, ids).to(torch.int16), (w * c["scale"]).float()


def _experts(c, x, ids, weights, layer):
    """Pairs sorted by expert and cut into blocks of one expert each; a block's products are one batched product."""
    t, k, n = x.shape[0], ids.shape[1], c["experts"]
    pairs = t * k
    block = max(1, min(128, pairs // n))
    e = ids.reshape(-1).long()
    e = torch.where(e < 0, n, e)  # empty slots last
    order = e.sort(stable=True).indices
    count = torch.zeros(n + 1, dtype=torch.long, device=x.device).scatter_add_(0, e, torch.ones_like(e))
    first = count.cumsum(0) - count
    need = (count[:n] + block - 1) // block
    ends = need.cumsum(0)
    total = min(pairs, pairs // block + n)
    b = torch.arange(total, device=x.device)
    of = torch.searchsorted(ends, b, right=True).clamp_(max=n - 1)
    at = (b - (ends - need)[of])[:, None] * block + torch.arange(block, device=x.device)
    real = (at < count[:n][of][:, None]) & (b < ends[-1])[:, None]
    pair = torch.where(real, order[(first[of][:, None] + at).clamp_(0, pairs - 1)], 0)
    rows = _quantised(x.float())[pair // k]
    (gq, gs), (uq, us), (dq, ds) = layer
    used = lambda q, s: _values(q.view(torch.uint8)[of].view(torch.float8_e4m3fn), s[of]).transpose(1, 2)  # noqa: E731
    g = torch.bmm(rows, used(gq, gs))
    h = g / (1.0 + torch.exp(-g)) * torch.bmm(rows, used(uq, us))
    h = _quantised(h.view(-1, h.shape[2])).view_as(h)
    y = torch.bmm(h, used(dq, ds)) * (weights.reshape(-1)[pair] * real)[:, :, None]
    slot = torch.zeros(pairs + 1, y.shape[2], device=x.device)
    slot[torch.where(real, pair, pairs).view(-1)] = y.view(-1, y.shape[2])
    return slot[:pairs].view(t, k, -1).sum(1).to(torch.bfloat16)


# ---- one pass ---------------------------------------------------------------------------------
def run(st):
    c, kind = st["c"], st["c"]["kind"]
    if not own:
        if kind == "logits":
            return st["x"].float() @ st["w"].T
        if kind == "route":
            ids, w = _route(c, st["x"], st["bias"])
            return dict(ids=ids, w=w)
        if kind == "matmul":
            return (_quantised(st["x"].float()) @ _values(st["q"], st["s"]).T).to(TYPES[c["y"]])
        return [_experts(c, x, ids, w, layer) for x, ids, w, layer in zip(st["x"], st["ids"], st["w"], st["layers"])]
    be, b = st["be"], st["b"]
    if kind == "logits":
        be.router_logits_device(st["kept"].handles[0], b["x"], c["t"], c["experts"], c["hidden"], b["out"], x_type=c["x"])
        return st["out"]
    if kind == "route":
        be.route_tokens_device(b["x"], c["t"], c["experts"], c["top_k"], b["ids"], b["w"], logits_type=c["logits"],
                               score=c["score"], d_bias=b.get("bias"), n_groups=c["groups"], top_groups=c["top_groups"],
                               group_best=c["best"], renormalise=c["renorm"], scale=c["scale"], d_status=b["status"])
        return dict(ids=st["ids"], w=st["w"])
    if kind == "matmul":
        be.f8_matmul_device(st["kept"].handles[0], b["x"], c["t"], b["out"], x_type=c["x"], y_type=c["y"])
        return st["out"]
    for i, kept in enumerate(st["handles"]):
        be.f8_experts_device(kept.handles[0], b["x"][i], c["t"], b["ids"][i], b["w"][i], c["top_k"], b["out"][i], x_type=c["x"],
                             y_type="bf16", d_status=b["status"])
    return st["out"]


# ---- the same from the definitions, in 64 bits ---------------------------------------------
def _e4m3_table():
    """The 256 values of e4m3: sign, 4 exponent bits (bias 7), 3 fraction bits; 0x7F is not a number."""
    b = np.arange(256)
    ex, fr = (b >> 3) & 15, b & 7
    v = np.where(ex == 0, fr / 8 * 2.0 ** -6, (1 + fr / 8) * 2.0 ** (ex - 7.0))
    v = np.where((b & 127) == 127, np.nan, v)
    return torch.from_numpy(np.where(b >= 128, -v, v)).to(DEV)


def _exact_matrix(q, s):
    w = _e4m3_table()[q.view(torch.uint8).long()]
    r, k = torch.arange(q.shape[0], device=DEV) // 128, torch.arange(q.shape[1], device=DEV) // 128
    return w * s.double()[r[:, None], k[None, :]]


def _exact_rows(x):
    """Rows after quantisation; scales are the f32 numbers that the format stores."""
    out = torch.zeros(x.shape, dtype=torch.float64, device=DEV)
    for at in range(0, x.shape[1], 128):
        v = x[:, at:at + 128].float()
        a = v.abs().amax(1, keepdim=True).double()
        s, inv = (a / 448).float().double(), (448 / a).float().double()
        z = (v.double() * inv).float().double()  # the product is a 32-bit one
        ulp = torch.exp2((torch.frexp(z).exponent - 1).clamp(min=-6).double() - 3)
        z = torch.clamp(torch.round(z / ulp) * ulp, -448, 448)
        out[:, at:at + 128] = torch.where(a < 2.0 ** -100, 0.0, z * s)
    return out


def _exact_route(c, lg, bias):
    lg = lg.double().cpu().numpy()
    b = np.zeros(lg.shape[1]) if bias is None else bias.double().cpu().numpy()
    out = np.zeros((lg.shape[0], c["top_k"]), np.float64)
    size = lg.shape[1] // c["groups"]
    for row, l in enumerate(lg):
        live = np.isfinite(l)
        if not live.any():
            continue
        p = np.zeros_like(l)
        p[live] = np.exp(l[live] - l[live].max()) if c["score"] == "softmax" else 1 / (1 + np.exp(-l[live]))
        if c["score"] == "softmax":
            p /= p.sum()
        v = np.where(live, p + b, -np.inf)
        if c["groups"] > 1:
            total = [sum(sorted((x for x in v[g * size:(g + 1) * size] if x > -np.inf), reverse=True)[:c["best"]])
                     if (v[g * size:(g + 1) * size] > -np.inf).any() else -np.inf for g in range(c["groups"])]
            for g in np.argsort([-x for x in total], kind="stable")[c["top_groups"]:]:
                v[g * size:(g + 1) * size] = -np.inf
        pick = [i for i in np.argsort(-v, kind="stable")[:c["top_k"]] if v[i] > -np.inf]
        w = p[pick]
        out[row, :len(pick)] = (w / w.sum() if c["renorm"] and w.sum() > 0 else w) * c["scale"]
    return dict(ids=None, w=out)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    c, kind = st["c"], st["c"]["kind"]
    if kind == "logits":
        return st["x"].double() @ st["w"].double().T
    if kind == "route":
        return _exact_route(c, st["x"], st["bias"])
    if kind == "matmul":
        return _exact_rows(st["x"]) @ _exact_matrix(st["q"], st["s"]).T
    got = []
    for x, ids, w, layer in zip(st["x"], st["ids"], st["w"], st["layers"]):
        rows, y = _exact_rows(x), torch.zeros(x.shape, dtype=torch.float64, device=DEV)
        for e in ids.unique().tolist():
            if e == NONE:
                continue
            t, k = (ids == e).nonzero(as_tuple=True)
            gate, up, down = (_exact_matrix(q[e], s[e]) for q, s in layer)
            g = rows[t] @ gate.T
            h = (g * torch.sigmoid(g) * (rows[t] @ up.T)).float()
            y.index_add_(0, t, w[t, k].double()[:, None] * (_exact_rows(h) @ down.T))
        got.append(y)
    return got


# ---- what a pass cannot do without ------------------------------------------------------------
_SIZE = {"f32": 4, "bf16": 2}


def work(case):
    c, t = case, case["t"]
    if c["kind"] == "logits":
        return dict(bytes=t * c["hidden"] * _SIZE[c["x"]] + 4 * c["experts"] * (c["hidden"] + t), flops=2.0 * t * c["hidden"] * c["experts"])
    if c["kind"] == "route":  # a score and its comparisons count as 10 operations
        return dict(bytes=t * c["experts"] * _SIZE[c["logits"]] + 6 * t * c["top_k"] + 4 * c["experts"] * c["bias"], flops=10.0 * t * c["experts"])
    if c["kind"] == "matmul":
        return dict(bytes=t * c["cols"] * _SIZE[c["x"]] + t * c["rows"] * _SIZE[c["y"]] + c["rows"] * c["cols"]
                    + 4 * _blocks(c["rows"]) * _blocks(c["cols"]), flops=2.0 * t * c["rows"] * c["cols"])
    n, size = c["layers"], 3.0 * c["hidden"] * c["width"]
    used = c["experts"] * (1 - (1 - min(1.0, c["top_k"] / c["experts"])) ** (t * (1 - c["empty"])))  # distinct experts, even routes
    return dict(bytes=n * (used * size + t * c["hidden"] * (_SIZE[c["x"]] + 2) + 6 * t * c["top_k"]),
                flops=n * 2.0 * t * (1 - c["empty"]) * c["top_k"] * size)
