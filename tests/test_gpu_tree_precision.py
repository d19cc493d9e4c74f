"""How many bits paged_tree_attention keeps of its probabilities, and what they depend on."""

import math

import pytest
import torch

from tests._tree import Case

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("ctx", [600, 5000])
def test_a_row_does_not_depend_on_its_neighbours(hip, dtype, D, ctx):
    """One query scaled up, whose maximum keeps rising: the other rows of the tile keep their bits."""
    c = Case([32, 3], [ctx, 40], 2, 2, D, dtype, seed=23)
    want = c.call()
    c.dq[5] *= 25
    got = c.call()
    others = [i for i in range(35) if i != 5]
    assert not torch.equal(got[5], want[5])
    assert torch.equal(got[others], want[others])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [64, 128, 256, 32])
@pytest.mark.parametrize("gap", [9.0, 12.0, 15.0, 18.0])
@pytest.mark.parametrize("ctx", [300, 3000])
def test_a_tail_below_a_sink_key_counts(hip, dtype, D, gap, ctx):
    """One key scores `gap` above all others; its value is 0, theirs 1.  A row's result is the tail's
    share, n e^-gap / (1 + n e^-gap) of the n other keys it sees.  Rounded are the result and, once
    each, the probabilities: half a step of the type (bf16 2^-8, fp16 2^-11, where an fp16
    probability is off by 2^-32 of the row's largest at least, a result by 2^-25), and the
    scores, exponentials and sums of n + 1 terms in fp32."""
    c = Case([20, 3], [ctx, 60], 4, 2, D, dtype, seed=3)
    c.dk.zero_()
    c.dv.fill_(1)
    c.dq.zero_()
    c.dq[:, :, 1] = 1
    for s in c.slots:
        c.dk[int(s[0]), :, 1], c.dv[int(s[0])] = 2 * gap, 0
    got = c.call(scale=0.5).double().cpu()
    at = 0
    for n, length, see in zip(c.q_lens, c.ctx, c.see):
        others = torch.from_numpy(see.sum(1)).double()[:, None, None] + (length - n - 1)
        tail = others * torch.exp(torch.tensor(-gap, dtype=torch.float64))
        want = tail / (1 + tail)
        half = torch.finfo(dtype).eps / 2
        # (the score 2 gap scale log2(e) and its exponential: gap 2^-22 and 2^-22 at most)
        bound = want * (2 * half * (1 + half) + (length + 4 * gap + 16) * 2.0 ** -24)
        if dtype == F16:
            bound = bound + others * 2.0 ** -32 + 2.0 ** -25
        err = (got[at:at + n] - want).abs()
        assert bool((err <= bound).all()), f"{float((err / bound).max()):.3g} of the bound"
        at += n


def _wide_bits(dtype, D, ctx, n, values):
    """n nodes of 3 heads over one KV head; keys 0 to 2 score 0, q0 and q1 and have the values
    `values`(p) in each dimension, p (rows, 3) their probabilities over the row's largest times
    some power of two; the others score -16 and have value 0.  Returns (got, want, size) per
    dimension, whose row is d % rows: the attention, and sum p |v| over sum p."""
    B, G, scale, f64 = 2, 3, 0.5, torch.float64
    g = torch.Generator().manual_seed(7)
    c = Case([n] * B, [ctx] * B, G, 1, D, dtype, seed=1, kind="chain")
    q = torch.zeros((n, G, D), dtype=f64)
    q[..., :2] = torch.rand((n, G, 2), generator=g) * 3 - 1.5
    q[..., 2] = 4
    q = q.to(dtype)
    c.dq.copy_(q.repeat(B, 1, 1))
    c.dk.zero_()
    c.dv.zero_()
    rows, ids = n * G, [torch.from_numpy(s).to(c.dk.device) for s in c.slots]
    p = (scale * (q.to(f64).view(rows, D)[:, :2] * 2)).exp()
    p = torch.cat((torch.ones(rows, 1, dtype=f64), p), 1)
    mine = torch.arange(D) % rows
    v = values(p[mine]).to(dtype)                             # (3, D)
    for s in ids:
        c.dk[s[1], 0, 0], c.dk[s[2], 0, 1] = 2, 2
        c.dk[s[3:], 0, 2] = -8
        c.dv[s[:3], 0] = v.to(c.dv.device)
    seen = ctx - n + 1 + torch.arange(n).repeat_interleave(G)
    total = (p.sum(1) + (seen - 3) * math.exp(-16))[mine]
    terms = p[mine] * v.to(f64).t()
    got = c.call(scale=scale).to(f64).cpu().view(B, rows, D)[:, mine, torch.arange(D)]
    return got, terms.sum(1) / total, terms.abs().sum(1) / total


@pytest.mark.parametrize("dtype,D", [(BF16, 256), (F32, 64), (F32, 256), (BF16, 32)])
@pytest.mark.parametrize("ctx,n", [(300, 5), (2000, 5), (2000, 60)])
def test_cancelling_sums_keep_24_bits(hip, dtype, D, ctx, n):
    """Where probabilities are fp32 (256-wide heads, fp32 caches, the general kernel), as in the
    other attention.  The values are chosen so that p0 v0 + p1 v1 + p2 v2 cancels to about 2^-18
    of its terms.  A score errs by the roundings of its exponent (below 2^-22 of p here) and of
    exp2 (2^-23), a sum of three by 2^-23: below 2^-21 in all, of sum p |v|.  16 bits of p would
    err by 2^-17."""
    def values(p):
        v0 = torch.ones(len(p), dtype=torch.float64)
        v1 = (-p[:, 0] / p[:, 1]).to(dtype).double()
        v2 = -(p[:, 0] + p[:, 1] * v1) / p[:, 2]
        return torch.stack((v0, v1, v2))
    got, want, size = _wide_bits(dtype, D, ctx, n, values)
    half = torch.finfo(dtype).eps / 2                         # (the output's own rounding)
    worst = float((((got - want).abs() - half * want.abs()) / size).max())
    assert worst <= 2.0 ** -20, f"2^{math.log2(worst):.2f}"


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("size,step", [(10, 1), (20, 8), (24, 8), (25, 4), (25, 8), (26, 8), (27, 16),
                                       (28, 32)])
@pytest.mark.parametrize("scale", [math.log(2.0), 1.0])
def test_large_scores(hip, dtype, D, size, step, scale):
    """Scores of 2^size and, from key 40 or 170 on, `step` more (both exact in fp32; a later one
    exceeds the first by a step of fp32 or a few): no operand overflows, and the weights are 1 and
    e^(scale step), whose exponent is off by a rounding of it and of log2(e) scale, 2^-23 of it
    each at most.  (The tile kernel: the general kernel and the fp32 tiles round scores first.)"""
    for turn in (40, 170):
        c = Case([6], [300], 4, 2, D, dtype, seed=size)
        c.dk.zero_()
        c.dq.zero_()
        first, second = (torch.from_numpy(s).to(c.dk.device)
                         for s in (c.slots[0][:turn], c.slots[0][turn:]))
        c.dq[:, :, 0], c.dq[:, :, 1] = 2.0 ** (size // 2), 1
        c.dk[:, :, 0] = 2.0 ** (size - size // 2)
        c.dk[second, :, 1] = step
        c.dv[first], c.dv[second] = 1.0, 0.0
        got = c.call(scale=scale).double().cpu()
        seen = torch.from_numpy(c.see[0].sum(1)).double()[:, None, None] + 300 - 6 - turn
        share = turn / (turn + seen * math.exp(scale * step))   # of the first keys, whose value is 1
        half = torch.finfo(dtype).eps / 2
        bound = share * (2 * half * (1 + half) + 2.0 ** -21 * step + 300 * 2.0 ** -24)
        if dtype == F16:
            # the running maximum is a multiple of fp32's step at that size, up to half of one above
            # what it stands for, and the end of fp16 as much nearer
            unit = 2.0 ** (math.floor(math.log2(2.0 ** size * scale * math.log2(math.e))) - 23)
            bound = bound + 2.0 ** -25 + turn * 2.0 ** (-31 + unit / 2) / (turn + seen)
        err = (got - share).abs()
        assert bool(torch.isfinite(got).all()), turn
        assert bool((err <= bound).all()), (turn, float((err / bound).max()))
