"""Windowed and quantised attention, and quantised rows, over caches whose rows lie past 4 GiB: the same
bits as over a small cache."""

import pytest
import torch

from tests._util import randn
from tests._window import Case

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
STRIDE, SLOTS = 1 << 16, 6 << 16          # bytes from slot to slot; 24 GiB with them


@pytest.fixture(scope="module")
def memory():
    buf = torch.empty((SLOTS, STRIDE), dtype=torch.uint8, device=DEV)
    yield buf
    del buf
    torch.cuda.empty_cache()


def _spread(memory, tensors):
    """Views (slots, heads, width) of memory, one for each tensor (S, heads, width), side by side in a
    slot; block i of a tensor is the view's block 3 i, counted from the end where i is odd.  Returns the
    views and the block numbers."""
    S = tensors[0].shape[0]
    n = S // 16
    ids = torch.tensor([SLOTS // 16 - 1 - 3 * i if i % 2 else 3 * i for i in range(n)], device=DEV)
    slots = (ids[:, None] * 16 + torch.arange(16, device=DEV)).reshape(-1)
    views, at = [], 0
    for t in tensors:
        es = t.element_size()
        view = torch.as_strided(memory.view(-1).view(t.dtype), (SLOTS, *t.shape[1:]),
                                (STRIDE // es, t.shape[2], 1), at // es)
        view[slots] = t[:16 * n]
        views.append(view)
        at += -(-t.shape[1] * t.shape[2] * es // 64) * 64
    return views, ids


@pytest.mark.parametrize("fmt,dtype", [(None, BF16), (None, F32), ("fp8", BF16), ("fp8", F32), ("fp4", F16)])
@pytest.mark.parametrize("q_lens,ctx,Hq,KVH,D", [
    ([1, 1], [900, 400], 8, 2, 128), ([5, 3], [900, 400], 8, 2, 64), ([30, 2], [700, 300], 4, 1, 128),
    ([150, 3], [700, 300], 4, 2, 128), ([40, 3], [700, 300], 4, 2, 256)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (200, 4)])
def test_attention(hip, memory, fmt, dtype, q_lens, ctx, Hq, KVH, D, window, sinks):
    c = Case(q_lens, ctx, Hq, KVH, D, dtype, window, sinks, seed=3, fmt=fmt)
    want = c.call()
    c.check(want)
    tensors = [c.dk, c.dks, c.dv, c.dvs] if fmt else [c.dk, c.dv]
    views, ids = _spread(memory, tensors)
    if fmt:
        c.dk, c.dks, c.dv, c.dvs = views
    else:
        c.dk, c.dv = views
    c.bt = torch.where(c.bt >= 0, ids[c.bt.clamp_min(0).long()].int(), c.bt)
    assert int(c.bt.max()) * 16 * STRIDE > 20 << 30
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert torch.equal(c.call(err=err), want) and int(err) == 0


def test_small_head_dims(hip, memory):
    """The general kernel."""
    c = Case([9, 2], [300, 80], 4, 2, 32, BF16, 100, 4, seed=3)
    want = c.call()
    (c.dk, c.dv), ids = _spread(memory, [c.dk, c.dv])
    c.bt = torch.where(c.bt >= 0, ids[c.bt.clamp_min(0).long()].int(), c.bt)
    assert torch.equal(c.call(), want)


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_rows(hip, memory, fmt, dtype):
    from dispec_amd.kv.quant_cache import quant_append, quant_gather
    T, H, D = 33, 2, 128
    width = D if fmt == "fp8" else D // 2
    near = [torch.zeros(48, H, w, dtype=torch.uint8, device=DEV) for w in (width, D // 32) * 2]
    far, ids = _spread(memory, near)
    k, v = randn((T, H, D), 1, dtype).to(DEV), randn((T, H, D), 2, dtype).to(DEV)
    slots = torch.arange(T, device=DEV)
    quant_append(*near, slots, k, v)
    there = ids[slots // 16] * 16 + slots % 16
    quant_append(*far, there, k, v)
    for a, b in zip(near, far):
        assert torch.equal(a[slots], b[there])
    for a, b in zip(quant_gather(*near, slots, dtype), quant_gather(*far, there, dtype)):
        assert torch.equal(a, b)
