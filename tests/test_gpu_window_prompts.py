"""Windowed and quantised attention of prompt chunks: tiles of many rows, more key chunks than a wave
looks up at a time, bad blocks, infinities and NaN beside them."""

import numpy as np
import pytest
import torch

from tests._util import f64
from tests._window import Case

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16 = torch.bfloat16, torch.float16
INF = float("inf")


def _reference(c, skip=()):
    """(o, A) as Case.reference's, a head at a time."""
    q = f64(c.q)
    o, A = np.zeros(q.shape), np.zeros(q.shape)
    at = 0
    for b, n in enumerate(c.q_lens):
        seen = torch.from_numpy(c.see[b].copy())
        for s, key in skip:
            if s == b:
                seen[:, key] = False
        some = seen.any(0)
        k, v = (torch.from_numpy(t[c.slots[b]]) for t in (c.k64, c.v64))
        k[~some], v[~some] = 0, 0
        for h in range(c.Hq):
            s = torch.from_numpy(q[at:at + n, h]) @ k[:, h // c.G].T * c.D ** -0.5
            s[~seen] = -INF
            p = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e300))
            p /= p.sum(-1, keepdim=True).clamp_min(1e-300)
            o[at:at + n, h] = (p @ v[:, h // c.G]).numpy()
            A[at:at + n, h] = (p @ v[:, h // c.G].abs()).numpy()
        at += n
    return o, A


@pytest.mark.parametrize("D,dtype,fmt,window,sinks", [
    (64, BF16, None, 0, 0), (128, F16, None, 4200, 70), (128, BF16, "fp8", 0, 0),
    (64, F16, "fp4", 4200, 130)])
def test_more_chunks_than_lanes(hip, D, dtype, fmt, window, sinks):
    """Tiles enough for the chip, so that each takes all of its 70 chunks."""
    c = Case([1200, 1100, 1200, 700], [4500, 4200, 4700, 4300], 13, 13, D, dtype, window, sinks,
             seed=D, fmt=fmt)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = c.call(err=err)
    assert int(err) == 0
    o, A = _reference(c)
    c.check(got, o, A)
    assert torch.equal(got, c.call())
    # a bad block that the second look-up finds
    c.bt[2, 4160 // 16] = 1 << 20
    got = c.call(err=err)
    assert int(err) > 0
    c.check(got, *_reference(c, [(2, k) for k in range(4160, 4176)]))


@pytest.mark.parametrize("fmt", [None, "fp8", "fp4"])
@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, BF16), (128, F16)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (260, 20), (40, 3)])
def test_bad_blocks(hip, D, dtype, fmt, window, sinks):
    c = Case([150, 140, 9], [700, 151, 400], 4, 2, D, dtype, window, sinks, seed=5, fmt=fmt)
    bad = {0: [0, 9, 35, 36, 37, 38, 43], 1: [0, 1, 9], 2: [24]}
    skip = []
    for b, blocks in bad.items():
        for i in blocks:
            c.bt[b, i] = 1 << 20
            skip += [(b, k) for k in range(16 * i, min(16 * i + 16, c.ctx[b]))]
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = c.call(err=err)
    assert int(err) > 0
    c.check(got, *_reference(c, skip))


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (260, 20), (40, 3)])
@pytest.mark.parametrize("holes", [(), (36, 41)])
def test_infinities(hip, D, dtype, window, sinks, holes):
    """To the rows that see their keys, whichever wave has them; beside blocks that have no id."""
    c = Case([150, 3], [700, 90], 4, 2, D, dtype, window, sinks, seed=6)
    for i in holes:
        c.bt[0, i] = 1 << 20
    keep = c.call()
    for key, x in ((2, INF), (300, -INF), (545, INF), (570, float("nan")), (630, -INF), (699, INF)):
        slot, d = int(c.slots[0][key]), key % D
        was = c.dv[slot, 1, d].clone()
        c.dv[slot, 1, d] = x
        got = c.call()
        c.dv[slot, 1, d] = was
        want = keep.clone()
        want[torch.from_numpy(c.see[0][:, key]).nonzero()[:, 0].to(DEV), 2:4, d] = x
        assert torch.equal(torch.nan_to_num(got, 1e4, 2e4, 3e4), torch.nan_to_num(want, 1e4, 2e4, 3e4)), key


@pytest.mark.parametrize("fmt", [None, "fp8"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (260, 20)])
def test_graph_of_two_calls_beside_eager_ones(hip, fmt, window, sinks):
    """Two captured calls of one graph, replayed on other lengths while eager calls run on a second
    stream; their workspaces are their own."""
    c = Case([150, 3], [1700, 900], 4, 2, 128, BF16, window, sinks, seed=8, fmt=fmt, hole=0)
    ctx = c.lens.clone()
    c.call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        one, two = c.call(), c.call(scale=0.25)
    side = torch.cuda.Stream()
    for step in range(4):
        c.lens.copy_(ctx - 40 * step)
        want = c.call(), c.call(scale=0.25)
        one.fill_(3.0)
        side.wait_stream(torch.cuda.current_stream())
        g.replay()
        with torch.cuda.stream(side):
            beside = [c.call() for _ in range(3)]
        torch.cuda.current_stream().wait_stream(side)
        for got in (one, *beside):
            assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want[0])), step
        assert torch.equal(torch.nan_to_num(two), torch.nan_to_num(want[1])), step


@pytest.mark.parametrize("fmt", [None, "fp4"])
@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, F16)])
def test_strides_and_rows_behind(hip, D, dtype, fmt):
    """q and out as parts of wider rows, heads between others; rows of no sequence stay."""
    c = Case([150, 0, 140], [400, 5, 333], 6, 2, D, dtype, 100, 7, seed=9, fmt=fmt)
    want = c.call()
    c.check(want, *_reference(c))
    q = torch.full((295, 8, 2 * D), float("nan"), dtype=dtype, device=DEV)
    q[:290, 1:7, D:] = c.dq
    out = torch.full((295, 7, D + 8), 5.0, dtype=dtype, device=DEV)
    got = c.call(q=q[:, 1:7, D:], out=out[:, 1:, :D])
    assert got.data_ptr() == out[:, 1:].data_ptr()
    assert torch.equal(got[:290], want)
    out[:290, 1:, :D] = 5.0
    assert (out == 5).all()
