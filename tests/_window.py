"""Windows, sinks and quantised caches for the tests: the formats and the attention in float64."""

from __future__ import annotations

import math

import numpy as np
import torch

from tests._util import f64, gen, randn

GROUP = 32
FP16_END = {"fp8": 61440.0, "fp4": 49152.0}
MOST = {"fp8": 448.0, "fp4": 6.0}


def numbers(fmt: str) -> list[float]:
    """What the codes without a sign stand for (e4m3: but for the last, which is no number)."""
    bits, bias, n = (3, 7, 127) if fmt == "fp8" else (1, 1, 8)
    out = []
    for c in range(n):
        e, m = c >> bits, c & ((1 << bits) - 1)
        out.append(math.ldexp(m + ((1 << bits) if e else 0), max(e, 1) - bias - bits))
    return out


def quantise(x: torch.Tensor, fmt: str):
    """(codes, scales) of rows (..., D), by the definition: search in the list of numbers."""
    a = f64(x)
    if x.dtype == torch.float16:
        a = np.where(np.isfinite(a), np.clip(a, -FP16_END[fmt], FP16_END[fmt]), a)
    g = a.reshape(*a.shape[:-1], -1, GROUP)
    odd = ~np.isfinite(g).all(-1)
    g = np.where(odd[..., None], 0.0, g)
    most = np.abs(g).max(-1)
    e = np.full(most.shape, -100)
    for k in range(-100, 118):
        e = np.where(most > MOST[fmt] * 2.0 ** k, k + 1, e)
    t = np.array(numbers(fmt))
    y = np.abs(g) / 2.0 ** e[..., None].astype(np.float64)
    y = np.minimum(y, MOST[fmt])
    up = np.minimum(np.searchsorted(t, y), len(t) - 1)
    down = np.maximum(up - 1, 0)
    far, near = t[up] - y, y - t[down]
    code = np.where((far < near) | ((far == near) & (up % 2 == 0)), up, down)
    sign = np.signbit(g)
    code = (code + sign * (128 if fmt == "fp8" else 8)).astype(np.uint8).reshape(a.shape)
    if fmt == "fp4":
        code = code[..., 0::2] | (code[..., 1::2] << 4)
    return torch.from_numpy(code), torch.from_numpy(np.where(odd, 255, e + 127).astype(np.uint8))


def values(code: torch.Tensor, scale: torch.Tensor, fmt: str) -> np.ndarray:
    """The float64 values that codes and scales stand for."""
    c, s = code.numpy().astype(np.int64), scale.numpy().astype(np.float64)
    if fmt == "fp4":
        c = np.stack([c & 15, c >> 4], -1).reshape(*c.shape[:-1], -1)
    t = np.array(numbers(fmt) + ([math.nan] if fmt == "fp8" else []))
    x = np.concatenate([t, -t])[c]
    s = np.where(s == 255, math.nan, 2.0 ** (s - 127))
    return x * np.repeat(s, GROUP, -1)


class Case:
    """A batch over a paged cache whose blocks lie anywhere.  Of blocks that no query of their
    sequence sees the table's entry is `hole`; rows that no query sees, and those of no sequence, are
    NaN.  fmt: a quantised cache (the rows' groups NaN)."""

    def __init__(self, q_lens, ctx, Hq, KVH, D, dtype, window=0, sinks=0, seed=0, bs=16, fmt=None,
                 hole=-7, device="cuda", spread=1.0):
        self.q_lens, self.ctx, self.bs, self.G = list(q_lens), list(ctx), bs, Hq // KVH
        self.Hq, self.KVH, self.D, self.dtype, self.fmt = Hq, KVH, D, dtype, fmt
        self.window, self.sinks = window, sinks
        need = [-(-c // bs) for c in ctx]
        blocks = sum(need) + 3
        perm = torch.randperm(blocks, generator=gen(seed)).tolist()
        bt = torch.full((len(ctx), max(need + [1])), hole, dtype=torch.int32)
        held = np.zeros(blocks * bs, dtype=bool)
        self.slots, self.see, at = [], [], 0
        for b, n in enumerate(need):
            ids = perm[at:at + n]
            at += n
            j = np.arange(ctx[b])
            pos = ctx[b] - q_lens[b] + np.arange(q_lens[b])[:, None]
            see = j <= pos
            if window:
                see &= (j > pos - window) | (j < sinks)
            self.see.append(see)
            slots = np.array(ids, dtype=np.int64)[j // bs] * bs + j % bs if n else j
            self.slots.append(slots)
            any_row = see.any(0)
            held[slots[any_row]] = True
            for i in range(n):
                if any_row[i * bs:(i + 1) * bs].any():
                    bt[b, i] = ids[i]
        k = randn((blocks * bs, KVH, D), seed + 1, dtype) * spread
        v = randn((blocks * bs, KVH, D), seed + 2, dtype)
        free = torch.from_numpy(~held)
        k[free] = float("nan")
        v[free] = float("nan")
        self.q = randn((sum(q_lens), Hq, D), seed + 3, dtype)
        self.max_q, self.max_ctx = max(q_lens), bt.shape[1] * bs
        cu = torch.tensor(np.concatenate([[0], np.cumsum(q_lens)]), dtype=torch.int32)
        self.cu, self.bt = cu.to(device), bt.to(device)
        self.lens = torch.tensor(ctx, dtype=torch.int32, device=device)
        self.dq = self.q.to(device)
        if fmt:
            (kc, ks), (vc, vs) = quantise(k, fmt), quantise(v, fmt)
            self.k64, self.v64 = values(kc, ks, fmt), values(vc, vs, fmt)
            self.dk, self.dks, self.dv, self.dvs = (t.to(device) for t in (kc, ks, vc, vs))
        else:
            self.k64, self.v64 = f64(k), f64(v)
            self.dk, self.dv = k.to(device), v.to(device)

    def call(self, cu="own", **kw):
        from dispec_amd.engine.hip_attn import paged_quant_attention, paged_window_attention
        args = dict(window=self.window, sinks=self.sinks, block_size=self.bs, max_q_len=self.max_q,
                    max_ctx=self.max_ctx)
        args.update(kw)
        cu = self.cu if isinstance(cu, str) else cu
        q = args.pop("q", self.dq)
        if self.fmt:
            return paged_quant_attention(q, self.dk, self.dks, self.dv, self.dvs, self.bt, cu,
                                         self.lens, self.G, **args)
        return paged_window_attention(q, self.dk, self.dv, self.bt, cu, self.lens, self.G, **args)

    def reference(self, scale=None, skip=()):
        """(o, A): the attention in float64, and sum_j p_j |v_j|, each (T, Hq, D).  skip: (b, key)
        pairs that count for nothing."""
        scale = self.D ** -0.5 if scale is None else scale
        q = f64(self.q)
        o, A = np.zeros(q.shape), np.zeros(q.shape)
        at = 0
        for b, n in enumerate(self.q_lens):
            seen = self.see[b].copy()
            for s, key in skip:
                if s == b:
                    seen[:, key] = False
            for i in range(n):
                keys = np.nonzero(seen[i])[0]
                if len(keys):
                    rows = self.slots[b][keys]
                    kk, vv = self.k64[rows], self.v64[rows]          # (keys, KVH, D)
                    qq = q[at + i].reshape(self.KVH, self.G, self.D)
                    s = np.einsum("khd,hgd->hgk", kk, qq) * scale
                    p = np.exp(s - s.max(-1, keepdims=True))
                    p /= p.sum(-1, keepdims=True)
                    o[at + i] = np.einsum("hgk,khd->hgd", p, vv).reshape(self.Hq, self.D)
                    A[at + i] = np.einsum("hgk,khd->hgd", p, np.abs(vv)).reshape(self.Hq, self.D)
            at += n
        return o, A

    def bound(self, o, A):
        """How far the output may be from o.  Half a step of the type for its rounding and, in 16
        bits, for each probability's (against the row sum of unrounded ones; an fp16 probability
        below 2^-14 of what it is held as rounds by 2^-25 at most).  In 32 bits: a score is a sum of D
        products, off by (D + 2) 2^-24 sum |q k| at most, which a probability follows; its exponential
        and the weights of the merged parts a few steps each, the sums over keys ctx steps."""
        half = torch.finfo(self.dtype).eps / 2
        k = float(np.nanmax(np.sqrt((self.k64 ** 2).sum(-1))))
        qk = float(np.sqrt((f64(self.q) ** 2).sum(-1)).max()) * k * self.D ** -0.5
        most = max(self.ctx + [1])
        f32 = 2.0 ** -24 * (2 * (self.D + 2) * qk + most + 64)
        out = half * np.abs(o) + f32 * A
        if self.dtype != torch.float32:
            out = out * (1 + 2 * half) + half * A * (1 + 2 * half)
        if self.dtype == torch.float16:
            out = out + 2.0 ** -25 * most * float(np.nanmax(np.abs(self.v64)))
        return out + 1e-30

    def check(self, got, o=None, A=None, what=""):
        if o is None:
            o, A = self.reference()
        err = np.abs(f64(got) - o)
        over = err / self.bound(o, A)
        assert np.isfinite(over).all(), f"{what}: not finite"
        assert over.max(initial=0.0) <= 1.0, f"{what}: {over.max():.3g} of the bound, {err.max():.3g}"
