"""Captured windowed and quantised attention replayed on new lengths: every row that a length makes
visible holds numbers, so each replay is held to the attention in float64 of its own lengths."""

import numpy as np
import pytest
import torch

from tests._util import randn
from tests._window import Case, quantise, values

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


class Live(Case):
    """A Case whose rows are all numbers and whose table is whole; `move` changes the lengths."""

    def __init__(self, q_lens, ctx, Hq, KVH, D, dtype, window, sinks, seed=0, fmt=None, device="cuda"):
        super().__init__(q_lens, ctx, Hq, KVH, D, dtype, window, sinks, seed=seed, fmt=fmt, device=device)
        for b, slots in enumerate(self.slots):
            ids = torch.from_numpy(slots[::self.bs] // self.bs).int()
            self.bt[b, :len(ids)] = ids.to(device)
        k, v = (randn((self.dk.shape[0], KVH, D), seed + i, dtype) for i in (5, 6))
        if fmt:
            (kc, ks), (vc, vs) = quantise(k, fmt), quantise(v, fmt)
            self.k64, self.v64 = values(kc, ks, fmt), values(vc, vs, fmt)
            for t, x in ((self.dk, kc), (self.dks, ks), (self.dv, vc), (self.dvs, vs)):
                t.copy_(x)
        else:
            self.k64, self.v64 = k.double().numpy(), v.double().numpy()
            self.dk.copy_(k)
            self.dv.copy_(v)

    def move(self, ctx):
        self.ctx, self.see = list(ctx), []
        for n, length in zip(self.q_lens, ctx):
            j, pos = np.arange(length), length - n + np.arange(n)[:, None]
            see = j <= pos
            if self.window:
                see &= (j > pos - self.window) | (j < self.sinks)
            self.see.append(see)
        self.lens.copy_(torch.tensor(self.ctx, dtype=torch.int32))


# (new tokens, contexts, tokens less a replay, query heads, KV heads, head_dim): decodes, few rows, up to
# 128, prompt chunks
BATCHES = [([1, 1, 1], [900, 500, 2000], 61, 8, 2, 128), ([2, 1, 3], [900, 500, 2000], 61, 8, 2, 64),
           ([30, 2], [1100, 400], 67, 4, 1, 128), ([150, 3], [1700, 900], 173, 4, 2, 128),
           ([40, 3], [900, 400], 67, 4, 2, 256)]
WINDOWS = [(0, 0), (300, 4), (70, 20)]


def _captured(f):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        f()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = f()
    return g, out


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,dtype", [(None, BF16), (None, F32), ("fp8", BF16), ("fp8", F32), ("fp4", F16)])
@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("window,sinks", WINDOWS)
def test_replays(hip, fmt, dtype, batch, window, sinks):
    q_lens, ctx, less, Hq, KVH, D = batch
    c = Live(q_lens, ctx, Hq, KVH, D, dtype, window, sinks, seed=9, fmt=fmt)
    g, out = _captured(c.call)
    for step in (0, 3, 1, 4):
        c.move([max(x - less * step, n) for x, n in zip(ctx, q_lens)])
        out.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        c.check(out, what=f"step {step}")
        assert torch.equal(out, c.call()), step


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [None, "fp8"])
@pytest.mark.parametrize("batch", [BATCHES[0], BATCHES[3]])
@pytest.mark.parametrize("window,sinks", WINDOWS[:2])
def test_two_graphs_and_eager_calls_at_once(hip, fmt, batch, window, sinks):
    """Two graphs of two calls each, replayed on two streams beside eager calls on a third: none uses
    another's workspace."""
    q_lens, ctx, less, Hq, KVH, D = batch
    cases = [Live(q_lens, ctx, Hq, KVH, D, BF16, window, sinks, seed=s, fmt=fmt) for s in (8, 18)]
    graphs = [_captured(lambda c=c: (c.call(), c.call(scale=0.25))) for c in cases]
    streams = [torch.cuda.Stream() for _ in range(3)]
    for step in range(4):
        for c, (_, outs) in zip(cases, graphs):
            c.move([x - less * step for x in ctx])
            for o in outs:
                o.fill_(float("nan"))
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
                g.replay()
        with torch.cuda.stream(streams[2]):
            beside = [c.call() for c in cases + cases]
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        for c, (_, (one, two)), eager in zip(cases + cases, graphs + graphs, beside):
            c.check(eager)
            assert torch.equal(eager, one)
            c.check(two, *c.reference(scale=0.25))


@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("window,sinks", WINDOWS)
def test_every_replay_attends_numbers(batch, window, sinks):
    """Computed here: the outputs that the replays are compared with are numbers, and other ones."""
    q_lens, ctx, less, Hq, KVH, D = batch
    c = Live(q_lens, ctx, Hq, KVH, D, BF16, window, sinks, seed=9, device="cpu")
    seen = []
    for step in (0, 1, 3, 4):
        c.move([max(x - less * step, n) for x, n in zip(ctx, q_lens)])
        o, _ = c.reference()
        assert np.isfinite(o).all() and not any(np.array_equal(o, x) for x in seen)
        seen.append(o)
