"""Attention layers in front of MoE layers, one sequence's cache for each.

A layer adds its attention to the residual rows x [t, H]:

    xn      = rmsnorm(x)                                     tqf_hip_rmsnorm_rows_device
    rows    = xn Wqkv^T, bf16: each query head with its      tqf_hip_f8_matmul_device
              gate, then the key heads, then the value heads
    q, k, v = norm and rotation of the heads, k and v into   tqf_hip_qk_rope_device
              the cache at the rows' positions
    y       = attention of q, times sigmoid(gate)            tqf_hip_attn_prompt_device, or
                                                             tqf_hip_attn_paged_device
    x      += y Wout^T                                       tqf_hip_f8_matmul_device,
                                                             tqf_hip_add_rows_device

The projections are e4m3 matrices with a scale for each block of 128 x 128. A
prompt in front of which there is nothing attends to its own rows; up to 8
rows behind what the cache holds attend over the cache. A row's slot is that
of its position, so rows behind a position that were put there for drafts
which were not accepted are written over by what comes next, and no row sees
them before.
"""
from __future__ import annotations

import numpy as np

from . import synth
from ._lib import F8_MAX_TOKENS, MAX_TOKENS
from .workloads import H

F8_BLOCK = 128


def f8_synthetic(rows: int, cols: int, seed: int) -> tuple[np.ndarray, np.ndarray]:
    """Seeded e4m3 bytes [rows, cols] and block scales: values of standard deviation cols^-1/2, in steps of all sizes."""
    rng = np.random.default_rng(seed)
    q = rng.integers(0, 256, size=(rows, cols), dtype=np.uint8)
    q[(q & 127) == 127] ^= 1  # NaN
    mags = np.arange(127)
    e, m = mags >> 3, mags & 7
    values = np.where(e == 0, m / 8.0 * 2.0 ** -6, (1.0 + m / 8.0) * 2.0 ** (e - 7.0))
    std = np.sqrt((values * values).mean())
    s = rng.uniform(0.8, 1.2, (-(-rows // F8_BLOCK), -(-cols // F8_BLOCK))) / (std * np.sqrt(cols))
    return q, s.astype(np.float32)


class AttentionLayers:
    """`n_layers` seeded attention layers of (query heads, key and value heads, head dimension), with a cache of
    `max_tokens` positions each (`cache`: "bf16" or "f8") in pages of `page`.  `rotary` elements of a head turn, by
    theta^(-2 i / rotary) a position.  One sequence: `forward` is told how many tokens the cache holds; `sequence` is
    whoever began the one that is there (None: none is whole)."""

    def __init__(self, be, n_layers: int, heads=(16, 2, 256), rotary: int = 64, theta: float = 1e7, gated: bool = True,
                 max_tokens: int = 4096, page: int = 64, cache: str = "bf16", seed: int = 0):
        nq, nk, d = heads
        if n_layers < 1 or max_tokens < 1:
            raise ValueError("AttentionLayers: at least one layer and one token")
        if rotary < 0 or rotary % 2 or rotary > d:
            raise ValueError("AttentionLayers: rotary is an even number of a head's elements")
        self.be, self.n_layers, self.heads, self.gated, self.max_tokens, self.page = be, n_layers, (nq, nk, d), gated, max_tokens, page
        self.max_prompt = min(max_tokens, F8_MAX_TOKENS)  # the projections' rows
        self.frequencies = [theta ** (-2.0 * i / rotary) for i in range(rotary // 2)]
        self.q_width = d * (2 if gated else 1)  # a query head with its gate
        self.width = nq * self.q_width + 2 * nk * d
        self.host, self.norms, self.q_norms, self.k_norms, self.qkv, self.out, self.caches = [], [], [], [], [], [], []
        self.rope, self._bufs, self.sequence = None, [], None
        try:
            self.rope = be.prepare_rope(self.frequencies) if rotary else None
            pages = -(-max_tokens // page)
            for layer in range(n_layers):
                s = seed + 1000 * layer
                norm, qn, kn = ((1.0 + 0.05 * synth.normal((n,), seed=s + 21 + i)).astype(np.float32) for i, n in enumerate((H, d, d)))
                wqkv, wout = f8_synthetic(self.width, H, s + 24), f8_synthetic(H, nq * d, s + 25)
                self.host.append(dict(norm=norm, q_norm=qn, k_norm=kn, qkv=wqkv, out=wout))
                self.norms.append(be.upload_f32(norm))
                self.q_norms.append(be.upload_f32(qn))
                self.k_norms.append(be.upload_f32(kn))
                self.qkv.append(be.upload_f8(*wqkv))
                self.out.append(be.upload_f8(*wout))
                self.caches.append(be.alloc_kv_cache(pages, nk, page, d, cache))
            # the sequence's pages, not in order; what a call needs of the counting numbers is a view of them
            self.table = np.random.default_rng(seed).permutation(pages).astype(np.int32)
            at = np.arange(max_tokens + 1, dtype=np.int32)
            self.d_pages, self.d_count = self._buf(self.table), self._buf(at)
            self.d_slots = self._buf(self.table[at[:-1] // page] * page + at[:-1] % page)
            rows = max(self.max_prompt, MAX_TOKENS)
            self.d_cu = self._buf(np.zeros(2, np.int32))
            self.d_xn, self.d_o = self._buf(4 * rows * H), self._buf(4 * rows * H)
            self.d_qkv, self.d_q, self.d_y = self._buf(2 * rows * self.width), self._buf(2 * rows * nq * d), self._buf(2 * rows * nq * d)
            self.d_k = self._buf(2 * rows * nk * d)
        except Exception:
            self.free()
            raise

    def _buf(self, what):
        self._bufs.append(self.be.alloc(what) if isinstance(what, int) else self.be.to_device(what))
        return self._bufs[-1]

    def forward(self, layer: int, d_x, t: int, at: int, d_status=None, trace: list | None = None) -> None:
        """d_x [t, H] += attention of the rows at positions at..at + t: all of a prompt (at = 0, up to `max_prompt`), or
        up to 8 rows behind the `at` tokens in the cache.  `trace`: host copies of the stages are added to it."""
        be, (nq, nk, d) = self.be, self.heads
        if t < 1 or at < 0 or at + t > self.max_tokens:
            raise ValueError(f"positions {at}..{at + t} of a cache of {self.max_tokens} tokens")
        if t > self.max_prompt:
            raise ValueError(f"at most {self.max_prompt} rows of a prompt")
        if at and t > MAX_TOKENS:
            raise ValueError(f"at most {MAX_TOKENS} rows behind the first of a sequence")
        x = be.read(d_x, np.float32, (t, H)).copy() if trace is not None else None
        be.rmsnorm_rows_device(d_x, t, H, self.norms[layer], self.d_xn)
        be.f8_matmul_device(self.qkv[layer], self.d_xn, t, self.d_qkv, y_type="bf16")
        w, q_width, kv_at = self.width, self.q_width, nq * self.q_width
        part = lambda first: be.view(self.d_qkv, 2 * first, self.d_qkv.nbytes - 2 * first)  # noqa: E731
        prompt = at == 0 and t > MAX_TOKENS  # a short one is as fast over the cache
        be.qk_rope_device(self.d_qkv, part(kv_at), part(kv_at + nk * d), t, self.heads, be.view(self.d_count, 4 * at, 4 * t), self.d_q,
                          d_k_out=self.d_k if prompt else None, x_type="bf16",
                          strides=((w, q_width), (w, d), (w, d)), q_norm=self.q_norms[layer], k_norm=self.k_norms[layer], rope=self.rope,
                          cache=self.caches[layer], d_slots=be.view(self.d_slots, 4 * at, 4 * t), d_status=d_status)
        gate = dict(d_gate=part(d), gate_strides=(w, q_width)) if self.gated else {}
        if prompt:
            be.copy_device(be.view(self.d_cu, 4, 4), be.view(self.d_count, 4 * t, 4), 4)
            be.attn_prompt_device(self.d_q, self.d_k, part(kv_at + nk * d), self.heads, self.d_cu, self.d_cu, 1, t, t, self.d_y,
                                  strides=(None, None, (w, d)), d_status=d_status, **gate)
        else:
            be.attn_paged_device(self.d_q, self.heads, 1, t, self.caches[layer], self.d_pages, len(self.table),
                                 be.view(self.d_count, 4 * (at + t), 4), self.d_y, d_status=d_status, **gate)
        be.f8_matmul_device(self.out[layer], self.d_y, t, self.d_o, x_type="bf16")
        be.add_rows_device(d_x, self.d_o, t * H, d_x)
        if trace is not None:
            read = lambda b, kind, *shape: be.read(b, kind, shape).copy()  # noqa: E731
            trace.append(dict(layer=layer, at=at, prompt=prompt, x=x, xn=read(self.d_xn, np.float32, t, H), rows=read(self.d_qkv, np.uint16, t, w),
                              q=read(self.d_q, np.uint16, t, nq, d), y=read(self.d_y, np.uint16, t, nq, d), o=read(self.d_o, np.float32, t, H),
                              out=read(d_x, np.float32, t, H), k=read(self.d_k, np.uint16, t, nk, d) if prompt else None,
                              cache=self.read_cache(layer)))

    def read_cache(self, layer: int):
        """Host copies of a layer's keys and values [pages, kv heads, page, head dimension] (bf16 bits, or e4m3 bytes with
        their scales)."""
        c, (_, nk, d) = self.caches[layer], self.heads
        shape = (c.n_pages, nk, self.page, d)
        kind = np.uint8 if c.type == "f8" else np.uint16
        out = [self.be.read(b, kind, shape).copy() for b in (c.d_k, c.d_v)]
        return out + ([self.be.read(b, np.float32, shape[:3]).copy() for b in (c.d_k_scales, c.d_v_scales)] if c.type == "f8" else [])

    def free(self) -> None:
        be = self.be
        for b in self._bufs:
            be.free(b)
        for t in self.norms + self.q_norms + self.k_norms:
            be.free_tensor(t)
        for m in self.qkv + self.out:
            be.free_weights(m)
        for c in self.caches:
            be.free_kv_cache(c)
        if self.rope is not None:
            be.free_rope(self.rope)
        self.rope, self._bufs = None, []
        self.norms, self.q_norms, self.k_norms, self.qkv, self.out, self.caches = [], [], [], [], [], []
