"""paged_tree_attention and tree_mask against the attention written out in float64."""

import random

import numpy as np
import pytest
import torch

from tests._tree import Case, ancestors, pack, random_parents
from tests._util import f64

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("parents", [True, False])
@pytest.mark.parametrize("q_lens", [[1], [5, 0, 33], [64, 1, 65], [300, 2]])
def test_tree_mask(hip, q_lens, parents):
    from dispec_amd.engine.hip_attn import tree_mask
    rng = random.Random(sum(q_lens))
    trees = [random_parents(n, rng, "tree" if parents else "chain") for n in q_lens]
    if parents and q_lens[0] > 3:
        trees[0][2] = -1     # a second root
        trees[0][3] = 3      # not an earlier node: a root too
    cu = _i32(np.concatenate([[0], np.cumsum(q_lens)]))
    flat = _i32([p for t in trees for p in t])
    got = tree_mask(flat if parents else None, cu, max(q_lens), num_tokens=sum(q_lens))
    assert torch.equal(got.cpu(), pack([ancestors(t) for t in trees], -(-max(q_lens) // 32)))
    assert torch.equal(got, tree_mask(flat if parents else None, cu, num_tokens=sum(q_lens)))


SHAPES = [(4, 2, 64), (4, 4, 128), (7, 1, 128), (6, 2, 256), (14, 2, 64)]
SMALL = [(4, 2, 32), (2, 1, 16), (3, 1, 8)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("Hq,KVH,D", SHAPES + SMALL)
@pytest.mark.parametrize("q_lens,ctx", [
    ([1], [1]), ([1, 1, 1], [1, 64, 300]),                 # single tokens
    ([5, 0, 17], [5, 40, 17]),                             # trees with no context before them
    ([8, 33, 1, 2], [70, 129, 513, 47]),                   # ends inside blocks and tiles
    ([64, 31], [64 + 192, 1000]),
    ([40, 130], [1111, 700]),
])
def test_trees(hip, dtype, Hq, KVH, D, q_lens, ctx):
    c = Case(q_lens, ctx, Hq, KVH, D, dtype, seed=D + len(ctx))
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = c.call(err=err)
    assert int(err) == 0
    c.check(got, what=f"{dtype} {Hq}/{KVH}x{D} {q_lens} {ctx}")
    assert torch.equal(got, c.call())                      # the same bits again


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["chain", "star"])
@pytest.mark.parametrize("D", [64, 128])
def test_chains_are_causal_and_stars_see_the_root(hip, dtype, kind, D):
    from dispec_amd.engine.hip_attn import paged_mq_attention
    c = Case([9, 40, 3], [200, 77, 3], 6, 2, D, dtype, seed=5, kind=kind)
    got = c.call()
    c.check(got, what=kind)
    if kind == "chain":
        o, A = c.reference()
        mq = paged_mq_attention(c.dq, c.dk, c.dv, c.bt, c.cu, c.lens, c.G, max_q_len=c.max_q,
                                max_ctx=c.max_ctx)
        c.check(mq, o, A, "paged_mq_attention")            # the same function


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("n,ctx", [(7, 7), (70, 70), (70, 300)])
def test_any_mask_and_rows_that_see_nothing(hip, dtype, D, n, ctx):
    """Masks that are no tree's: rows without any bit (zeros where there is no context either),
    bits above the diagonal, bits past the tree (which count for nothing)."""
    rng = np.random.default_rng(n + D)
    see = [rng.random((n, n)) < 0.2, rng.random((3, 3)) < 0.5]
    see[0][1] = False
    see[0][n - 1] = False
    see[1][:] = False
    c = Case([n, 3], [ctx, 3], 4, 2, D, dtype, seed=n, see=see)
    c.mask[0, -1] |= -(1 << 31) if n % 32 else 0           # node 31 or 95: past the tree
    got = c.call()
    c.check(got, what="any mask")
    assert bool((got[n:] == 0).all())
    if ctx == n:
        assert bool((got[1] == 0).all()) and bool((got[n - 1] == 0).all())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [64, 128, 256, 32])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("ctx", [50, 900])
def test_nonfinite_values_reach_the_rows_that_see_them(hip, dtype, D, bad, ctx):
    """V of one node (and K, where it is NaN) spoilt: its rows' outputs are what the formula gives,
    the others what they were."""
    n = 40
    c = Case([n, 6], [ctx, 300], 4, 2, D, dtype, seed=17)
    want = c.call()
    node = 11
    slot = int(c.slots[0][ctx - n + node])
    c.dv[slot, 0, 3] = bad
    got = c.call()
    sees = np.zeros(n + 6, dtype=bool)
    sees[:n] = c.see[0][:, node]
    hit = torch.from_numpy(sees).to(DEV)
    ref = want.clone()
    ref[hit, :2, 3] = bad                                  # the 2 heads of KV head 0
    assert torch.equal(got.isnan(), ref.isnan())
    assert torch.equal(got.nan_to_num(7.0), ref.nan_to_num(7.0))
    if bad != bad:
        c.dv[slot, 0, 3] = 0.0
        c.dk[slot, 1, 5] = bad
        got = c.call()
        assert bool(got[hit, 2:].isnan().all())
        assert torch.equal(got[~hit, 2:], want[~hit, 2:])


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (BF16, 128), (F16, 256), (F32, 64), (BF16, 32)])
@pytest.mark.parametrize("bs", [1, 4, 16, 64])
def test_block_sizes_strides_and_out(hip, dtype, D, bs):
    """Blocks of any size, q as the rows of a fused projection, caches with padded rows and a slot
    stride, an `out` whose rows behind the last sequence stay."""
    c = Case([5, 34], [61, 250], 6, 2, D, dtype, seed=bs, bs=bs)
    T = c.dq.shape[0]
    qkv = torch.full((T, 10, D), float("nan"), dtype=dtype, device=DEV)
    qkv[:, :6] = c.dq
    c.dq = qkv[:, :6]
    wide = torch.full((2, c.k.shape[0], 3, D), float("nan"), dtype=dtype, device=DEV)
    wide[0, :, :2], wide[1, :, :2] = c.dk, c.dv
    c.dk, c.dv = wide[0, :, :2], wide[1, :, :2]
    c.check(c.call(), what=f"bs {bs}")
    out = torch.full((T + 4, 8, D), 3.0, dtype=dtype, device=DEV)
    assert c.call(out=out[:T, 1:7]).data_ptr() == out[0, 1].data_ptr()
    c.check(out[:T, 1:7], what="out")
    assert bool((out[T:] == 3).all()) and bool((out[:, 0] == 3).all()) and bool((out[:, 7] == 3).all())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_rows_off_16_bytes(hip, dtype, D):
    """Caches and queries whose rows start at any element."""
    c = Case([20, 3], [90, 400], 4, 2, D, dtype, seed=9)
    off = []
    for t in (c.dq, c.dk, c.dv):
        flat = torch.empty(t.shape[0] * t.shape[1] * (D + 1) + 1, dtype=dtype, device=DEV)
        view = flat[1:].view(t.shape[0], t.shape[1], D + 1)[..., :D]
        view.copy_(t)
        off.append(view)
    c.dq, c.dk, c.dv = off
    out = torch.empty_like(c.dq)
    c.check(c.call(out=out), what="unaligned")


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (BF16, 128), (F16, 256), (F32, 64), (BF16, 16)])
@pytest.mark.parametrize("scale", [0.0, 0.3, -0.2, 2.0])
def test_scales(hip, dtype, D, scale):
    c = Case([12, 1], [200, 33], 4, 2, D, dtype, seed=3)
    c.q, c.dq = c.q / 4, c.dq / 4
    o, A = c.reference(scale)
    got = c.call(scale=scale)
    # (the scores are at most |scale| sqrt(D) times those that the bound takes, 2 sqrt(D) here)
    err = np.abs(f64(got) - o) / (c.bound(o, A) + 2.0 ** -24 * 64 * (c.D + 2) * c.D ** 0.5 * A)
    assert np.isfinite(err).all() and err.max() <= 1, err.max()


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (F16, 128), (BF16, 256), (F32, 64), (BF16, 32)])
def test_bad_lengths_and_blocks(hip, dtype, D):
    """Lengths that do not fit are counted once and give zeros; ids outside the pool are counted,
    their keys count for nothing."""
    c = Case([6, 4, 9, 20], [100, 64, 200, 333], 4, 2, D, dtype, seed=4)
    good = c.call()
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    lens = c.lens.clone()
    lens[1], lens[2] = 3, c.max_ctx + 1                    # fewer tokens than nodes, past the table
    keep, c.lens = c.lens, lens
    got = c.call(err=err)
    assert int(err) == 2
    assert bool((got[6:19] == 0).all())
    assert torch.equal(got[:6], good[:6]) and torch.equal(got[19:], good[19:])
    c.lens = keep
    skip = []
    for b, j, bad in ((0, 0, -1), (2, 5, c.k.shape[0] // c.bs), (3, 20, 2 ** 30), (3, 3, -2 ** 31)):
        c.bt[b, j] = bad
        skip += [(b, key) for key in range(j * 16, min(j * 16 + 16, c.ctx[b]))]
    err.zero_()
    got = c.call(err=err)
    assert int(err) >= 4
    o, A = c.reference(skip=skip)
    c.check(got, o, A, "bad blocks")


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (F16, 64), (F32, 64)])
def test_more_nodes_than_the_bound(hip, dtype, D):
    """Of a longer tree the first max_q_len rows are computed (and see what their masks say)."""
    c = Case([40, 5], [300, 90], 4, 2, D, dtype, seed=6)
    out = torch.full_like(c.dq, 9.0)
    want = c.call()
    c.call(max_q_len=32, out=out)
    o, A = c.reference()
    for rows in (slice(0, 32), slice(40, 45)):
        err = np.abs(f64(out[rows]) - o[rows]) / c.bound(o, A)[rows]
        assert err.max() <= 1
    assert bool(torch.isfinite(want).all())


@pytest.mark.parametrize("dtype,Hq,KVH,D", [(BF16, 32, 8, 128), (F16, 28, 4, 128), (BF16, 14, 2, 64),
                                            (F32, 14, 2, 64), (BF16, 8, 8, 256)])
def test_long_contexts(hip, dtype, Hq, KVH, D):
    """Work that is cut into many parts and merged; some rows are looked at, all are finite."""
    q_lens, ctx = [64, 1, 30], [9001, 4111, 700]
    c = Case(q_lens, ctx, Hq, KVH, D, dtype, seed=8)
    got = f64(c.call())
    assert np.isfinite(got).all()
    for b, rows in ((0, (0, 17, 63)), (1, (0,)), (2, (29,))):
        at = sum(q_lens[:b])
        for i in rows:
            for h in (0, Hq - 1):
                seen = np.ones(ctx[b], dtype=bool)
                seen[ctx[b] - q_lens[b]:] = c.see[b][i]
                sl = c.slots[b][seen]
                kk, vv = f64(c.k)[sl, h // c.G], f64(c.v)[sl, h // c.G]
                s = kk @ f64(c.q)[at + i, h] * D ** -0.5
                p = np.exp(s - s.max())
                o, A = p @ vv / p.sum(), p @ np.abs(vv) / p.sum()
                assert (np.abs(got[at + i, h] - o) <= c.bound(o, A)).all(), (b, i, h)


def test_offsets_past_32_bits(hip):
    """Blocks whose rows lie more than 2^31 elements into the pool."""
    KVH, D, bs, n, ctx = 2, 128, 16, 10, 75
    slots = 2 ** 31 // (KVH * D) + 64 * bs
    c = Case([n], [ctx], 4, KVH, D, BF16, seed=21)
    big = [torch.empty((slots, KVH, D), dtype=BF16, device=DEV) for _ in range(2)]
    ids = [slots // bs - 1 - 3 * j for j in range(-(-ctx // bs))]
    at = torch.tensor([ids[j // bs] * bs + j % bs for j in range(ctx)], device=DEV)
    assert int(at.min()) * KVH * D > 2 ** 31 - 2 ** 16
    old = torch.from_numpy(c.slots[0]).to(DEV)
    want = c.call()
    big[0][at], big[1][at] = c.dk[old], c.dv[old]
    c.dk, c.dv = big
    c.bt[0, :len(ids)] = _i32(ids)
    assert torch.equal(c.call(), want)


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (F32, 64)])
def test_other_streams_and_graphs(hip, dtype, D):
    """A call on another stream, and one captured and replayed with other lengths, inputs and masks,
    between eager calls."""
    from dispec_amd.engine.hip_attn import tree_mask
    c = Case([16, 5], [900, 64], 6, 2, D, dtype, seed=13)
    d = Case([3, 18], [500, 700], 6, 2, D, dtype, seed=14)
    want = c.call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = c.call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    # static buffers; the trees are masks made inside the graph
    q = torch.zeros((21, 6, D), dtype=dtype, device=DEV)
    par = torch.full((21,), -1, dtype=torch.int32, device=DEV)
    cu, lens = torch.zeros_like(c.cu), torch.zeros_like(c.lens)
    width = max(c.bt.shape[1], d.bt.shape[1])
    bt = torch.zeros((2, width), dtype=torch.int32, device=DEV)
    kv = torch.zeros((2, max(len(c.k), len(d.k)), 2, D), dtype=dtype, device=DEV)
    from dispec_amd.engine.hip_attn import paged_tree_attention

    def body():
        mask = tree_mask(par, cu, 18)
        return paged_tree_attention(q, kv[0], kv[1], bt, cu, lens, mask, 3, max_q_len=18,
                                    max_ctx=width * 16)

    def load(x):
        q[:len(x.dq)].copy_(x.dq)
        par[:len(x.dq)].copy_(_i32([p for t in x.parents for p in t]))
        cu.copy_(x.cu)
        lens.copy_(x.lens)
        bt.zero_()
        bt[:, :x.bt.shape[1]].copy_(x.bt)
        kv[0, :len(x.k)].copy_(x.dk)
        kv[1, :len(x.k)].copy_(x.dv)

    load(c)
    body()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = body()
    for x in (c, d, c, d):
        load(x)
        eager = body()
        graph.replay()
        torch.cuda.synchronize()
        n = len(x.dq)
        assert torch.equal(out[:n], eager[:n])
        x.check(out[:n], what="replay")


def test_a_shared_workspace(hip):
    """One workspace for the layers of a forward, of any content; a small one is not used."""
    from dispec_amd.engine.hip_attn import tree_workspace
    c = Case([30, 7], [3000, 150], 8, 2, 128, BF16, seed=2)
    want = c.call()
    ws = tree_workspace(2, 8, 2, 128, c.max_q, c.max_ctx, DEV)
    if ws is not None:
        ws.fill_(float("nan"))
        for _ in range(3):
            assert torch.equal(c.call(workspace=ws), want)
    tiny = torch.zeros(4, device=DEV)
    assert torch.equal(c.call(workspace=tiny), want) and bool((tiny == 0).all())


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (F16, 128)])
def test_runs_longer_than_the_ids_held(hip, dtype, D):
    """Contexts so long, and so many, that a workgroup's part of one is longer than the block ids it
    holds at a time.  The tables name a few blocks again and again: a slot's weight in 64 bits is
    its count times its exponential."""
    from dispec_amd.engine.hip_attn import paged_tree_attention
    B, H, bs, n, ctx, blocks = 16, 8, 16, 3, 150_001, 40
    g = torch.Generator().manual_seed(31)
    k, v = (torch.randn(blocks * bs, H, D, generator=g).to(dtype).to(DEV) for _ in range(2))
    q = torch.randn(B * n, H, D, generator=g).to(dtype).to(DEV)
    width = -(-ctx // bs)
    bt = torch.randint(0, blocks, (B, width), generator=g, dtype=torch.int32)
    cu = torch.arange(0, B * n + 1, n, dtype=torch.int32, device=DEV)
    lens = torch.full((B,), ctx, dtype=torch.int32, device=DEV)
    mask = torch.tensor([[1], [3], [5]] * B, dtype=torch.int32, device=DEV)
    got = f64(paged_tree_attention(q, k, v, bt.to(DEV), cu, lens, mask, 1, block_size=bs, max_q_len=n,
                                   max_ctx=ctx))
    kk, vv, qq = f64(k), f64(v), f64(q)
    half = torch.finfo(dtype).eps / 2
    f32 = 2.0 ** -24 * (2 * (D + 2) * np.abs(qq).max() * np.abs(kk).max() * D ** 0.5 + ctx + 64)
    pos = np.arange(ctx)
    for b in range(B):
        slots = bt[b].numpy()[pos // bs].astype(np.int64) * bs + pos % bs
        base = np.bincount(slots[:ctx - n], minlength=blocks * bs).astype(np.float64)
        for i, nodes in enumerate(((0,), (0, 1), (0, 2))):
            count = base.copy()
            for a in nodes:
                count[slots[ctx - n + a]] += 1
            for h in range(H):
                s = kk[:, h] @ qq[b * n + i, h] * D ** -0.5
                p = count * np.exp(s - s.max())
                o, A = p @ vv[:, h] / p.sum(), p @ np.abs(vv[:, h]) / p.sum()
                bound = half * np.abs(o) + f32 * A
                bound = bound * (1 + 2 * half) + half * A * (1 + 2 * half)
                if dtype == F16:
                    bound = bound + 2.0 ** -25 * ctx * np.abs(vv).max()
                assert (np.abs(got[b * n + i, h] - o) <= bound).all(), (b, i, h)


@pytest.mark.parametrize("dtype,KVH,G,D,top", [(BF16, 8, 1, 64, 500), (BF16, 8, 2, 64, 1700),
                                               (F16, 8, 1, 128, 1300), (BF16, 2, 3, 256, 900)])
def test_many_sequences(hip, dtype, KVH, G, D, top):
    """More tiles than workgroups fit the chip: each has several, some of them cut; sequences
    without nodes and with a few tokens among them."""
    rng = random.Random(top)
    B = 600 // KVH if D < 256 else 140
    ctx = [rng.choice((1, 2, 17, rng.randint(1, top), rng.randint(top // 2, top))) for _ in range(B)]
    ctx[rng.randrange(B)] = top
    q_lens = [min(c, rng.choice((0, 1, 1, 2, 5))) for c in ctx]
    c = Case(q_lens, ctx, KVH * G, KVH, D, dtype, seed=top)
    c.check(c.call(), what=f"{B} sequences")


@pytest.mark.parametrize("seed", range(12))
def test_random_batches(hip, seed):
    """Shapes, lengths, block sizes and masks at random."""
    rng = random.Random(900 + seed)
    dtype = rng.choice((BF16, F16))
    D, KVH, G = rng.choice((64, 64, 128, 128, 256)), rng.choice((1, 2, 3)), rng.choice((1, 2, 5, 7, 8))
    B, bs = rng.randint(1, 7), rng.choice((16, 16, 32, 128))
    q_lens, ctx = [], []
    for _ in range(B):
        n = rng.choice((0, 1, rng.randint(2, 20), rng.randint(20, 100)))
        q_lens.append(n)
        ctx.append(n + rng.choice((0, 0, rng.randint(0, 64), rng.randint(0, 3000))))
    ctx = [max(x, 1) for x in ctx]
    if not sum(q_lens):
        q_lens[0] = 1
    masks = np.random.default_rng(seed)
    see = [masks.random((n, n)) < 0.5 for n in q_lens] if seed % 3 == 0 else None
    c = Case(q_lens, ctx, KVH * G, KVH, D, dtype, seed=seed, bs=bs, see=see)
    out = torch.full((c.dq.shape[0] + 3, *c.dq.shape[1:]), 7.0, dtype=dtype, device=DEV)
    c.check(c.call(out=out[:-3]), what=f"{dtype} {KVH}x{G}x{D} {q_lens} {ctx} blocks of {bs}")
    assert bool((out[-3:] == 7.0).all())
