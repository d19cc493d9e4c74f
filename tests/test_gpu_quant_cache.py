"""Rows into a quantised cache and back, bit by bit against the formats written out."""

import numpy as np
import pytest
import torch

from tests._util import f64, gen, randn
from tests._window import quantise, values

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _pools(L, S, H, D, fmt):
    width = D if fmt == "fp8" else D // 2
    shape, scales = (L, S, H, width), (L, S, H, D // 32)
    return [torch.full(s, 77, dtype=torch.uint8, device=DEV) for s in (shape, scales, shape, scales)]


def _rows(shape, seed, dtype):
    """Rows of all magnitudes, with zeros, halves between codes, and the type's ends."""
    x = torch.randn(shape, generator=gen(seed)) * torch.exp2(
        torch.randint(-20, 12, shape[:-1] + (1,), generator=gen(seed + 1)).float())
    x[..., ::7] = (x[..., ::7] * 64).round() / 64
    x.view(-1)[:5] = torch.tensor([0.0, -0.0, torch.finfo(dtype).max, -torch.finfo(dtype).max,
                                   torch.finfo(dtype).smallest_normal])
    flat = x.view(-1, shape[-1])
    flat[1 % len(flat)] = 0.0
    flat[2 % len(flat)] = torch.finfo(dtype).smallest_normal
    for i, p in enumerate((1, 3, 5, 7, 9, 11, 13, 15)):
        flat[3 % len(flat), i] = p / 8.0     # halves between codes beside a 6 and a 448
    flat[3 % len(flat), 20] = 6.0
    if len(flat) > 4:
        flat[4, :] = torch.arange(shape[-1]) * 2.0 + 200
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("L,T,H,D", [(1, 1, 1, 32), (1, 33, 8, 128), (3, 50, 2, 64), (2, 7, 3, 96),
                                     (1, 300, 2, 256)])
def test_round_trip(hip, dtype, fmt, L, T, H, D):
    from dispec_amd.kv.quant_cache import quant_append, quant_gather
    S = T + 5
    pools = _pools(L, S, H, D, fmt)
    k, v = _rows((L, T, H, D), 1, dtype), _rows((L, T, H, D), 2, dtype)
    slots = torch.randperm(S, generator=gen(3))[:T]
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    quant_append(*pools, slots.to(DEV), k.to(DEV), v.to(DEV), err=err)
    rest = torch.ones(S, dtype=torch.bool)
    rest[slots] = False
    for x, codes, scales in ((k, *pools[:2]), (v, *pools[2:])):
        want = quantise(x, fmt)
        codes, scales = codes.cpu(), scales.cpu()
        assert torch.equal(scales[:, slots], want[1])
        # (-0 and 0 are one number)
        assert np.array_equal(values(codes[:, slots], scales[:, slots], fmt), values(*want, fmt))
        assert (codes[:, rest] == 77).all() and (scales[:, rest] == 77).all()
    for out_type in (dtype, F32):
        got = quant_gather(*pools, slots.to(DEV), out_type, err=err)
        for x, g in zip((k, v), got):
            want = torch.from_numpy(values(*quantise(x, fmt), fmt)).to(out_type)
            assert bool(torch.isfinite(g).all())
            assert torch.equal(g.cpu(), want), f"{out_type}"
    assert int(err) == 0


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
def test_every_code_reads_back(hip, fmt):
    """All codes under all scales, in the three types (fp16: rounded, infinite past its range)."""
    from dispec_amd.kv.quant_cache import quant_gather
    code = torch.arange(256, dtype=torch.uint8)
    code = code[(code & 127) != 127] if fmt == "fp8" else code
    code = torch.cat([code, code[:(-len(code)) % 32]])
    scale = torch.arange(27, 246, dtype=torch.uint8)
    kc = code.view(1, 1, -1).expand(len(scale), 1, -1).contiguous()
    ks = scale.view(-1, 1, 1).expand(-1, 1, kc.shape[2] * (1 if fmt == "fp8" else 2) // 32).contiguous()
    want = torch.from_numpy(values(kc, ks, fmt))
    for dtype in (BF16, F16, F32):
        k, v = quant_gather(kc.to(DEV), ks.to(DEV), kc.to(DEV), ks.to(DEV),
                            torch.arange(len(scale), device=DEV), dtype)
        assert torch.equal(k.cpu(), want.to(dtype)) and torch.equal(k, v)


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_groups_without_a_scale(hip, dtype, fmt):
    """An infinity or NaN makes its group NaN, and no other; numbers past 2^118 M end there."""
    from dispec_amd.kv.quant_cache import quant_append, quant_gather
    x = randn((4, 1, 64), 1, dtype)
    x[0, 0, 5], x[1, 0, 40], x[2, 0, 63] = float("inf"), float("nan"), -float("inf")
    pools = [p[0] for p in _pools(1, 4, 1, 64, fmt)]
    slots = torch.arange(4, device=DEV)
    quant_append(*pools, slots, x.to(DEV), x.to(DEV))
    k, v = quant_gather(*pools, slots, dtype)
    want = torch.from_numpy(values(*quantise(x, fmt), fmt)).to(dtype)
    assert torch.isnan(want[0, 0, :32]).all() and torch.isnan(want[1:3, 0, 32:]).all()
    assert torch.equal(torch.isnan(k.cpu()), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(k.cpu()), torch.nan_to_num(want)) and torch.equal(
        torch.nan_to_num(k), torch.nan_to_num(v))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strided_rows(hip, dtype):
    """k and v as views of a fused projection, and at odd offsets."""
    from dispec_amd.kv.quant_cache import quant_append
    T, H, D = 9, 2, 64
    for off in (0, 1):
        x = randn((T, 4 * H * D + off), 1, dtype).to(DEV)[:, off:].view(T, 4 * H, D) if off == 0 else \
            randn((T, 4 * H * D + 3), 1, dtype).to(DEV)[:, off:off + 4 * H * D].unflatten(1, (4 * H, D))
        k, v = x[:, 2:2 + H], x[:, 5:5 + H]
        a, b = ([p[0] for p in _pools(1, T, H, D, "fp8")] for _ in "ab")
        slots = torch.arange(T, device=DEV)
        quant_append(*a, slots, k, v)
        quant_append(*b, slots, k.contiguous(), v.contiguous())
        assert all(torch.equal(p, r) for p, r in zip(a, b))


def test_slots_outside_the_pool(hip):
    from dispec_amd.kv.quant_cache import quant_append, quant_gather
    pools = _pools(2, 8, 2, 64, "fp8")
    before = [p.clone() for p in pools]
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    x = randn((2, 3, 2, 64), 1).to(DEV)
    quant_append(*pools, torch.tensor([-1, 8, 3], device=DEV), x, x, err=err)
    assert int(err) == 2
    for p, q in zip(pools, before):
        p[:, 3] = 77
        assert torch.equal(p, q)
    quant_gather(*pools, torch.tensor([0, 1 << 40], device=DEV), err=err)
    assert int(err) == 3


def _cache(L=2, blocks=12, bs=16, H=2, D=64, dtype=BF16, fmt="fp8"):
    from dispec_amd.kv.quant_cache import QuantPagedKVCache
    return QuantPagedKVCache(L, blocks, bs, H, D, dtype, DEV, format=fmt)


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_cache(hip, dtype, fmt):
    """write, gather, export, import, block copies and forks."""
    c = _cache(dtype=dtype, fmt=fmt)
    assert c.memory_bytes() < 0.53 * 2 * 2 * 12 * 16 * 2 * 64 * (2 if fmt == "fp8" else 1.1)
    ids = [7, 2, 9]
    k, v = randn((2, 40, 2, 64), 1, dtype).to(DEV), randn((2, 40, 2, 64), 2, dtype).to(DEV)
    c.import_contiguous(ids, k, v)
    kk, vv = (torch.from_numpy(values(*quantise(x.cpu(), fmt), fmt)).to(dtype).to(DEV) for x in (k, v))
    got = c.export_contiguous(ids, 40)
    assert torch.equal(got[0], kk) and torch.equal(got[1], vv)
    got = c.gather(1, c.context_slots(ids, 40))
    assert torch.equal(got[0], kk[1]) and torch.equal(got[1], vv[1])
    c.write(0, c.context_slots([4], 3), k[0, :3], v[0, :3])
    assert torch.equal(c.gather(0, c.context_slots([4], 3))[0], kk[0, :3])
    # two sequences, one of no tokens
    flat = c.export_batch([(ids, 40), ([4], 0), ([7], 5)])
    assert flat[2] == [0, 40, 40, 45]
    assert torch.equal(flat[0][:80].view(2, 40, 2, 64), kk)
    assert torch.equal(flat[1][80:].view(2, 5, 2, 64), vv[:, :5])
    d = _cache(dtype=dtype, fmt=fmt)
    d.import_batch([[1, 3, 5], [], [8]], flat[0], flat[1], flat[2])
    assert torch.equal(d.export_contiguous([1, 3, 5], 40)[0], kk)    # what was exported stays as it is
    # blocks as they are, one into one and one into many
    d.copy_blocks_from(c, [7, 2], [0, 6])
    assert torch.equal(d.export_contiguous([0, 6], 32)[1], vv[:, :32])
    d.copy_blocks([(0, 9), (0, 10), (0, 11)])
    for b in (9, 10, 11):
        assert torch.equal(d.key_scale[:, b * 16:b * 16 + 16], c.key_scale[:, 7 * 16:8 * 16])
        assert torch.equal(d.export_contiguous([b], 16)[0], kk[:, :16])
    assert torch.equal(c.export_contiguous(ids, 1)[0], kk[:, :1])
    c.check_errors()
    d.check_errors()


def test_commit_path(hip):
    c = _cache()
    k = randn((2, 16, 2, 64), 3).to(DEV)
    c.import_contiguous([5], k, k)
    was = c.export_contiguous([5], 16)[0]
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    c.commit_path(i32(5).view(1, 1), i32(0, 6), i32(16), i32(0, 3, 5, -1).view(1, 4), i32(2))
    now = c.export_contiguous([5], 16)[0]
    assert torch.equal(now[:, 11], was[:, 13]) and torch.equal(now[:, 12], was[:, 15])
    assert torch.equal(now[:, :11], was[:, :11]) and torch.equal(now[:, 13:], was[:, 13:])


def test_graph(hip):
    from dispec_amd.kv.quant_cache import quant_append, quant_gather
    pools = [p[0] for p in _pools(1, 64, 2, 128, "fp8")]
    x = randn((5, 2, 128), 1).to(DEV)
    slots = torch.arange(5, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        quant_append(*pools, slots, x, x)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        quant_append(*pools, slots, x, x)
        k, v = quant_gather(*pools, slots)
    for step in range(4):
        x.copy_(randn((5, 2, 128), 10 + step).to(DEV))
        slots.add_(7)
        g.replay()
        torch.cuda.synchronize()
        want = torch.from_numpy(values(*quantise(x.cpu(), "fp8"), "fp8")).to(BF16)
        assert torch.equal(k.cpu(), want) and torch.equal(v.cpu(), want)
        assert torch.equal(quant_gather(*pools, slots)[0], k)
