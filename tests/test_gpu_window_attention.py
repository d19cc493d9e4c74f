"""paged_window_attention and paged_quant_attention against the attention written out in float64.
Rows that no query sees are NaN, and blocks that none sees have no id."""

import pytest
import torch

from tests._window import Case

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32

SHAPES = [(4, 2, 64), (4, 4, 128), (7, 1, 128), (6, 2, 256), (14, 2, 64)]
SMALL = [(4, 2, 32), (2, 1, 16), (3, 1, 8)]
BATCHES = [
    ([1], [1]), ([1, 1, 1], [1, 64, 300]),                 # single tokens
    ([5, 0, 17], [5, 40, 17]),                             # no context before the new tokens
    ([8, 33, 1, 2], [70, 129, 513, 47]),                   # ends inside blocks and tiles
    ([40, 130], [1111, 700]),
]
WINDOWS = [(0, 0), (1, 0), (16, 4), (100, 0), (64, 64), (130, 70), (5000, 3)]


def _run(c, what):
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = c.call(err=err)
    assert int(err) == 0, what
    c.check(got, what=what)
    assert torch.equal(got, c.call()), what                # the same bits again


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("Hq,KVH,D", SHAPES + SMALL)
@pytest.mark.parametrize("window,sinks", WINDOWS)
def test_windows(hip, dtype, Hq, KVH, D, window, sinks):
    for i, (q_lens, ctx) in enumerate(BATCHES):
        c = Case(q_lens, ctx, Hq, KVH, D, dtype, window, sinks, seed=D + i)
        _run(c, f"{q_lens} {ctx}")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("Hq,KVH,D", SHAPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (16, 4), (130, 70)])
def test_quantised(hip, dtype, fmt, Hq, KVH, D, window, sinks):
    for i, (q_lens, ctx) in enumerate(BATCHES):
        c = Case(q_lens, ctx, Hq, KVH, D, dtype, window, sinks, seed=D + i, fmt=fmt)
        _run(c, f"{q_lens} {ctx}")


@pytest.mark.parametrize("fmt", [None, "fp8", "fp4"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_long(hip, dtype, fmt, D):
    """Many chunks a tile, several tiles a head, parts that a merge joins."""
    for window, sinks in ((0, 0), (700, 5)):
        c = Case([300, 1, 7], [2900, 4001, 1500], 4, 2, D, dtype, window, sinks, seed=D, fmt=fmt)
        _run(c, f"window {window}")


@pytest.mark.parametrize("fmt", [None, "fp8", "fp4"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("bs", [16, 32, 128])
def test_block_sizes(hip, dtype, fmt, bs):
    for window, sinks in ((0, 0), (40, 4), (200, 130)):
        _run(Case([9, 1, 70], [77, 600, 300], 4, 2, 64, dtype, window, sinks, seed=bs, bs=bs, fmt=fmt),
             f"window {window}")


@pytest.mark.parametrize("bs", [1, 8])
def test_small_blocks(hip, bs):
    _run(Case([9, 1], [77, 300], 4, 2, 64, BF16, 40, 4, seed=bs, bs=bs), "small blocks")


@pytest.mark.parametrize("fmt", [None, "fp8"])
@pytest.mark.parametrize("D,dtype", [(128, BF16), (128, F32), (64, F16), (32, BF16)])
def test_one_query_a_sequence_without_offsets(hip, D, dtype, fmt):
    if fmt and D == 32:
        pytest.skip("a quantised cache has heads of 64 and more")
    ctx = [1, 17, 900, 64, 2000]
    for window, sinks in ((0, 0), (33, 2), (600, 4)):
        c = Case([1] * 5, ctx, 8, 2, D, dtype, window, sinks, seed=5, fmt=fmt)
        c.check(c.call(cu=None))
        # a sequence without a context: zeros, not counted; a bad one: zeros, counted
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        c.lens[0], c.lens[3] = 0, c.max_ctx + 1
        out = c.call(cu=None, err=err, out=torch.full_like(c.dq, 9.0))
        assert int(err) == 1 and not out[0].any() and not out[3].any()
        # (the others' parts are cut elsewhere now: the same to rounding)
        keep = [1, 2, 4]
        o, A = c.reference()
        c.check(out[keep], o[keep], A[keep])


@pytest.mark.parametrize("fmt", [None, "fp8", "fp4"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strides(hip, dtype, fmt):
    """q and out as views of wider tensors, a layer of a larger pool with heads apart."""
    c = Case([6, 1, 40], [100, 300, 41], 4, 2, 64, dtype, 50, 4, seed=2, fmt=fmt)
    want = c.call()
    T, es = c.dq.shape[0], 16
    wide = torch.zeros((T, 6, 64 + es), dtype=dtype, device=DEV)
    wide[:, 1:5, :64] = c.dq
    out = torch.full((T, 6, 64 + es), 7.0, dtype=dtype, device=DEV)
    assert torch.equal(c.call(q=wide[:, 1:5, :64], out=out[:, 1:5, :64]), want)
    assert (out[:, 0] == 7).all() and (out[:, :, 64:] == 7).all() and (out[:, 5] == 7).all()

    def spaced(t, pad):
        big = torch.zeros((t.shape[0], t.shape[1] + 1, t.shape[2] + pad), dtype=t.dtype, device=DEV)
        big[:, :t.shape[1], :t.shape[2]] = t
        return big[:, :t.shape[1], :t.shape[2]]

    c.dk, c.dv = spaced(c.dk, 16), spaced(c.dv, 16)
    if fmt:
        c.dks, c.dvs = spaced(c.dks, 1), spaced(c.dvs, 1)
    assert torch.equal(c.call(), want)


def test_rows_off_alignment(hip):
    """Rows that no 16-byte load reaches, a negative scale: the general kernel."""
    c = Case([6, 1, 40], [100, 300, 41], 4, 2, 64, BF16, 50, 4, seed=2)
    wide = torch.zeros((c.dq.shape[0], 4, 65), dtype=BF16, device=DEV)
    wide[:, :, 1:] = c.dq
    c.check(c.call(q=wide[:, :, 1:]))
    c.check(c.call(scale=-0.1), *c.reference(scale=-0.1))
    c.check(c.call(scale=0.0), *c.reference(scale=0.0))


@pytest.mark.parametrize("fmt", [None, "fp8", "fp4"])
@pytest.mark.parametrize("dtype,D", [(BF16, 128), (F16, 64), (F32, 64), (BF16, 32)])
def test_bad_lengths_and_blocks(hip, dtype, D, fmt):
    if fmt and D == 32:
        pytest.skip("a quantised cache has heads of 64 and more")
    c = Case([3, 2, 4, 1], [60, 40, 200, 90], 4, 2, D, dtype, 48, 4, seed=1, fmt=fmt)
    good = c.call()
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    c.lens[1] = 1                     # fewer tokens than queries
    got = c.call(err=err)
    assert int(err) == 1
    assert not got[3:5].any() and torch.equal(got[:3], good[:3]) and torch.equal(got[5:], good[5:])
    # a block id outside the cache: its keys count for nothing
    c = Case([3, 2, 4, 1], [60, 40, 200, 90], 4, 2, D, dtype, 48, 4, seed=1, fmt=fmt)
    c.bt[2, 11] = 1 << 20             # keys 176 .. 191
    err.zero_()
    got = c.call(err=err)
    assert int(err) > 0
    c.check(got, *c.reference(skip=[(2, k) for k in range(176, 192)]))
    # no key left: zeros
    c.bt.fill_(-1)
    assert not c.call().any()


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (F16, 64), (F32, 64), (F32, 128), (BF16, 256), (BF16, 32)])
def test_infinities_reach_the_rows_that_see_them(hip, dtype, D):
    inf = float("inf")
    c = Case([70, 3], [300, 90], 4, 2, D, dtype, 33, 4, seed=D)
    keep = c.call()
    for key, x in ((2, inf), (231, -inf), (260, inf), (299, inf), (240, float("nan"))):
        d = key % D
        c.dv[int(c.slots[0][key]), 1, d] = x
        got = c.call()
        want = keep.clone()
        rows = torch.from_numpy(c.see[0][:, key]).nonzero()[:, 0].to(DEV)
        want[rows, 2:4, d] = x
        assert torch.equal(torch.nan_to_num(got, 1e4, 2e4, 3e4), torch.nan_to_num(want, 1e4, 2e4, 3e4)), key
        c.dv[int(c.slots[0][key]), 1, d] = float(c.v64[int(c.slots[0][key]), 1, d])


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_a_group_of_nan(hip, dtype, fmt):
    """A group whose scale is 255 is NaN to the rows that see its key, and to no others."""
    c = Case([70, 3], [300, 90], 4, 2, 64, dtype, 33, 4, seed=3, fmt=fmt)
    keep = c.call()
    slot = int(c.slots[0][250])
    c.dvs[slot, 0, 1] = 255
    got = c.call()
    rows = torch.from_numpy(c.see[0][:, 250]).nonzero()[:, 0].to(DEV)
    nan = torch.zeros_like(keep, dtype=torch.bool)
    nan[rows, :2, 32:] = True
    assert torch.equal(torch.isnan(got), nan)
    assert torch.equal(got[~nan], keep[~nan])
    # in K: a row that sees it is NaN throughout
    c.dvs[slot, 0, 1] = 127
    keep = c.call()
    c.dks[slot, 0, 0] = 255
    got = c.call()
    nan = torch.zeros_like(keep, dtype=torch.bool)
    nan[rows, :2] = True
    assert torch.equal(torch.isnan(got), nan) and torch.equal(got[~nan], keep[~nan])


@pytest.mark.parametrize("fmt", [None, "fp8", "fp4"])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_large_scores(hip, dtype, fmt):
    """Scores of thousands: the running maximum follows them, nothing overflows."""
    c = Case([20, 1], [300, 200], 4, 2, 64, dtype, 90, 4, seed=4, fmt=fmt, spread=200.0)
    got = c.call()
    assert bool(torch.isfinite(got).all())
    c.check(got)


def test_rows_behind_the_last_sequence_stay(hip):
    for fmt in (None, "fp8"):
        c = Case([3, 2], [60, 40], 4, 2, 64, BF16, 48, 4, seed=1, fmt=fmt)
        q = torch.cat([c.dq, torch.full((4, 4, 64), float("nan"), dtype=BF16, device=DEV)])
        out = torch.full_like(q, 5.0)
        c.call(q=q, out=out)
        assert (out[5:] == 5).all()
        c.check(out[:5])


def test_more_queries_than_the_bound(hip):
    """Of a sequence with more than max_q_len queries the first max_q_len rows are computed."""
    c = Case([9, 2], [60, 40], 4, 2, 64, BF16, 20, 2, seed=1)
    want = c.call()
    got = c.call(max_q_len=5, out=torch.full_like(c.dq, 3.0))
    assert torch.equal(got[:5], want[:5]) and torch.equal(got[9:], want[9:])
    assert (got[5:9] == 3).all()


@pytest.mark.parametrize("fmt", [None, "fp8"])
def test_streams_and_workspaces(hip, fmt):
    from dispec_amd.engine.hip_attn import window_workspace
    c = Case([4, 1], [4000, 3000], 8, 2, 128, BF16, 0, 0, seed=7, fmt=fmt)
    want = c.call()
    ws = window_workspace(2, 8, 2, 128, c.max_q, c.max_ctx, "cuda", format=fmt)
    assert ws is not None
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = c.call(workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    assert torch.equal(c.call(workspace=ws[:10]), want)    # too small: the call takes its own


@pytest.mark.parametrize("fmt", [None, "fp8", "fp4"])
def test_graph(hip, fmt):
    """Captured calls replay on new lengths, beside eager work."""
    c = Case([2, 1, 3], [900, 500, 2000], 8, 2, 64, BF16, 300, 4, seed=9, fmt=fmt, hole=0)
    ctx = c.lens.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.call()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = c.call()
    for step in range(4):
        c.lens.copy_(ctx - step * 7)
        out.fill_(3.0)
        g.replay()
        torch.cuda.synchronize()
        eager = c.call()
        assert torch.equal(torch.nan_to_num(out), torch.nan_to_num(eager)), step
