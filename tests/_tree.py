"""Drafted trees for the tests: random shapes, and the operators written out in float64."""

from __future__ import annotations

import random

import numpy as np
import torch

from tests._util import f64, gen, randn


def random_parents(n: int, rng: random.Random, kind: str = "tree") -> list[int]:
    """Parents of n nodes, each before its child; node 0 is the root."""
    if kind == "chain":
        return list(range(-1, n - 1))
    if kind == "star":
        return ([-1] + [0] * (n - 1))[:n]
    return ([-1] + [rng.randrange(max(0, i - 6), i) for i in range(1, n)])[:n]


def ancestors(parents: list[int]) -> np.ndarray:
    """(n, n) bool: node i sees node a (itself and its ancestors)."""
    n = len(parents)
    see = np.zeros((n, n), dtype=bool)
    for i, p in enumerate(parents):
        if 0 <= p < i:
            see[i] = see[p]
        see[i, i] = True
    return see


def pack(see: list[np.ndarray], words: int) -> torch.Tensor:
    """(sum n, words) int32 mask rows of the given visibility matrices."""
    out = np.zeros((sum(len(s) for s in see), words), dtype=np.uint32)
    at = 0
    for s in see:
        for i in range(len(s)):
            for a in np.nonzero(s[i])[0]:
                out[at + i, a >> 5] |= np.uint32(1) << np.uint32(a & 31)
        at += len(s)
    return torch.from_numpy(out.view(np.int32))


class Case:
    """A batch of trees over a paged cache whose blocks lie anywhere; slots that no key of the
    batch holds are NaN.  q_lens[b] of ctx[b] tokens are the nodes (0 of them: no row)."""

    def __init__(self, q_lens, ctx, Hq, KVH, D, dtype, seed=0, bs=16, kind="tree", see=None,
                 device="cuda"):
        rng = random.Random(seed)
        self.q_lens, self.ctx, self.bs, self.G = list(q_lens), list(ctx), bs, Hq // KVH
        self.Hq, self.KVH, self.D, self.dtype = Hq, KVH, D, dtype
        need = [-(-c // bs) for c in ctx]
        blocks = sum(need) + 3
        perm = torch.randperm(blocks, generator=gen(seed)).tolist()
        bt = torch.zeros((len(ctx), max(need + [1])), dtype=torch.int32)
        self.slots, at = [], 0
        for b, n in enumerate(need):
            ids = perm[at:at + n]
            at += n
            bt[b, :n] = torch.tensor(ids, dtype=torch.int32)
            j = np.arange(ctx[b])
            self.slots.append(np.array(ids, dtype=np.int64)[j // bs] * bs + j % bs if n
                              else np.zeros(0, dtype=np.int64))
        held = np.zeros(blocks * bs, dtype=bool)
        for s in self.slots:
            held[s] = True
        self.k = randn((blocks * bs, KVH, D), seed + 1, dtype)
        self.v = randn((blocks * bs, KVH, D), seed + 2, dtype)
        self.k[torch.from_numpy(~held)] = float("nan")
        self.v[torch.from_numpy(~held)] = float("nan")
        self.q = randn((sum(q_lens), Hq, D), seed + 3, dtype)
        self.parents = [random_parents(n, rng, kind) for n in q_lens]
        self.see = see if see is not None else [ancestors(p) for p in self.parents]
        self.max_q, self.max_ctx = max(q_lens), bt.shape[1] * bs
        self.mask = pack(self.see, max(1, -(-self.max_q // 32))).to(device)
        self.cu = torch.tensor(np.concatenate([[0], np.cumsum(q_lens)]), dtype=torch.int32)
        self.cu, self.bt = self.cu.to(device), bt.to(device)
        self.lens = torch.tensor(ctx, dtype=torch.int32, device=device)
        self.dk, self.dv, self.dq = (t.to(device) for t in (self.k, self.v, self.q))

    def call(self, **kw):
        from dispec_amd.engine.hip_attn import paged_tree_attention
        args = dict(block_size=self.bs, max_q_len=self.max_q, max_ctx=self.max_ctx)
        args.update(kw)
        return paged_tree_attention(self.dq, self.dk, self.dv, self.bt, self.cu, self.lens,
                                    self.mask, self.G, **args)

    def reference(self, scale=None, skip=()):
        """(o, A): the attention in float64, and sum_j p_j |v_j|, each (T, Hq, D).  skip: (b, key)
        pairs that count for nothing."""
        scale = self.D ** -0.5 if scale is None else scale
        k, v, q = f64(self.k), f64(self.v), f64(self.q)
        o = np.zeros(q.shape)
        A = np.zeros(q.shape)
        at = 0
        for b, (n, c) in enumerate(zip(self.q_lens, self.ctx)):
            seen = np.ones((n, c), dtype=bool)
            if n:
                seen[:, c - n:] = self.see[b]
            for s, key in skip:
                if s == b:
                    seen[:, key] = False
            for h in range(self.Hq):
                kk, vv = k[self.slots[b], h // self.G], v[self.slots[b], h // self.G]
                for i in range(n):
                    keys = np.nonzero(seen[i])[0]
                    if not len(keys):
                        continue
                    s = kk[keys] @ q[at + i, h] * scale
                    p = np.exp(s - s.max())
                    o[at + i, h] = p @ vv[keys] / p.sum()
                    A[at + i, h] = p @ np.abs(vv[keys]) / p.sum()
            at += n
        return o, A

    def bound(self, o, A):
        """How far the output may be from o.  Half a step of the type for its rounding and, in 16
        bits, for each probability's (against the row sum of unrounded ones; an fp16 probability
        below 2^-14 rounds by 2^-25 at most).  In 32 bits: a score is a sum of D products, off by
        (D + 2) 2^-24 sum |q k| at most, which a probability follows; its exponential and the
        weights of the merged parts a few steps each, the sums over keys ctx steps."""
        half = torch.finfo(self.dtype).eps / 2
        qk = float(np.abs(f64(self.q)).max()) * float(np.nanmax(np.abs(f64(self.k)))) * self.D ** 0.5
        most = max(self.ctx + [1])
        f32 = 2.0 ** -24 * (2 * (self.D + 2) * qk + most + 64)
        out = half * np.abs(o) + f32 * A
        if self.dtype != torch.float32:
            out = out * (1 + 2 * half) + half * A * (1 + 2 * half)
        if self.dtype == torch.float16:
            out = out + 2.0 ** -25 * most * float(np.nanmax(np.abs(f64(self.v))))
        return out + 1e-30

    def check(self, got, o=None, A=None, what=""):
        if o is None:
            o, A = self.reference()
        err = np.abs(f64(got) - o)
        over = err / self.bound(o, A)
        assert np.isfinite(over).all(), f"{what}: not finite"
        assert over.max(initial=0.0) <= 1.0, f"{what}: {over.max():.3g} of the bound, {err.max():.3g}"
