"""How many bits paged_window_attention and paged_quant_attention keep of their probabilities: all of
fp32's where a head has 256 dims, q is fp32 or the general kernel runs, as in the other attention of
those shapes; elsewhere (16-bit q, heads of 64 and 128) one operand of q's type.

A bound of the worst case lets a lost bit pass; the mean over a batch does not.  A rounding to nearest
is off by at most half a step, half |x|, spread evenly: by half |x| / sqrt(3) in the root of the mean
square, roundings of different numbers independent of each other.  With o = sum_j p_j v_j (sum_j p_j =
1), A = sum_j p_j |v_j| and

    sigma^2 = half^2 o^2                                 the output
            + half^2 sum_j (p_j v_j)^2                   where probabilities are one 16-bit operand
            + (2^-24 (sqrt(D) + sqrt(ctx) + 8) A)^2      scores and sums in fp32, a random walk of
                                                         as many steps; exponentials, weights

the mean square of err / sigma is 1/3 at most, its root 0.578; over N outputs it strays by about
1 / sqrt(N) of that.  The limit is 0.62, N 10000 and more."""

import math

import numpy as np
import pytest
import torch

from tests._util import f64
from tests._window import Case

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
LIMIT = 0.62
# (query heads, KV heads, head_dim, new tokens, contexts): few rows a KV head, up to 128, more
SHAPES = [(14, 2, 64, [5, 9], [300, 900]), (8, 2, 128, [8, 12], [500, 1200]),
          (8, 4, 256, [20, 9], [400, 700]), (8, 2, 256, [27, 9], [400, 700]),
          (4, 1, 256, [60, 2], [700, 90]), (16, 4, 128, [30, 3], [600, 200]),
          (4, 2, 64, [150, 3], [700, 90]), (4, 2, 128, [150, 3], [700, 90]),
          (16, 4, 32, [20, 9], [400, 700])]
WINDOWS = [(0, 0), (200, 4)]


def one_operand(dtype, D):
    return dtype != F32 and D in (64, 128)


def attend(c, p_type=None):
    """(o, sum (p v)^2, A, ctx), each (T, Hq, D) but ctx, in 64 bits; p_type: the probabilities,
    over the row's largest, rounded to it, the sum unrounded."""
    q = f64(c.q)
    o, sq, A = (np.zeros(q.shape) for _ in range(3))
    ctx, at = np.zeros((len(q), 1, 1)), 0
    for b, (n, length) in enumerate(zip(c.q_lens, c.ctx)):
        some = c.see[b].any(0)
        seen, slots = c.see[b][:, some], c.slots[b][some]
        ctx[at:at + n] = length
        for h in range(c.Hq):
            kk, vv = c.k64[slots, h // c.G], c.v64[slots, h // c.G]
            s = np.where(seen, q[at:at + n, h] @ kk.T * c.D ** -0.5, -np.inf)
            p = np.exp(s - s.max(1, keepdims=True))
            total = p.sum(1, keepdims=True)
            if p_type is not None:
                p = torch.from_numpy(p).to(p_type).double().numpy()
            p = p / total
            o[at:at + n, h], A[at:at + n, h] = p @ vv, p @ np.abs(vv)
            sq[at:at + n, h] = p ** 2 @ vv ** 2
        at += n
    return o, sq, A, ctx


def rms(c, got, exact):
    o, sq, A, ctx = exact
    half = torch.finfo(c.dtype).eps / 2
    var = (half * o) ** 2 + (2.0 ** -24 * (c.D ** 0.5 + ctx ** 0.5 + 8) * A) ** 2
    if one_operand(c.dtype, c.D):
        var = var + half ** 2 * sq
    assert o.size >= 10000
    return float(np.sqrt(((got - o) ** 2 / var).mean()))


def _case(shape, dtype, window, sinks, fmt, device="cuda"):
    Hq, KVH, D, q_lens, ctx = shape
    if fmt and D == 32:
        pytest.skip("a quantised cache has heads of 64 and more")
    return Case(q_lens, ctx, Hq, KVH, D, dtype, window, sinks, seed=31, fmt=fmt, device=device)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("fmt", [None, "fp8", "fp4"])
def test_mean_error(hip, dtype, shape, window, sinks, fmt):
    c = _case(shape, dtype, window, sinks, fmt)
    got = rms(c, f64(c.call()), attend(c))
    assert got <= LIMIT, got


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("dtype,narrower", [(F32, F16), (F16, BF16), (BF16, torch.float8_e4m3fn)])
def test_the_limit_tells_a_lost_type(shape, dtype, narrower, window, sinks):
    """Computed here: with the probabilities' own type the error is within the limit, with the next
    narrower one (where they are fp32: q's) it is not."""
    c = _case(shape, dtype, window, sinks, None, device="cpu")
    exact = attend(c)

    def simulated(p_type):
        return f64(torch.from_numpy(attend(c, p_type)[0]).to(dtype))

    own = dtype if one_operand(dtype, c.D) else F32
    assert rms(c, simulated(own), exact) <= LIMIT
    if own == F32 and dtype != F32:
        narrower = dtype
    assert rms(c, simulated(narrower), exact) > LIMIT


@pytest.mark.gpu
@pytest.mark.parametrize("ctx,n,window", [(300, 5, 0), (2000, 5, 0), (2000, 40, 0), (2000, 5, 900),
                                          (2000, 40, 900)])
def test_cancelling_sums_keep_24_bits(hip, ctx, n, window):
    """bf16, heads of 256.  Three keys, sinks under a window, score 0, q0 and q1; their values are
    chosen in dimension d for row d % rows so that p0 v0 + p1 v1 + p2 v2 cancels to about 2^-18 of
    its terms; the other keys score -16 and have value 0.  A score errs by the roundings of its
    exponent (below 2^-22 of p here) and of exp2 (2^-23), a sum of three by 2^-23: below 2^-21 in
    all, of sum p |v|.  16 bits of p would err by 2^-17."""
    B, G, D, scale, d64 = 2, 3, 256, 0.5, torch.float64
    g = torch.Generator().manual_seed(7)
    c = Case([n] * B, [ctx] * B, G, 1, D, BF16, window, 4 if window else 0, seed=1)
    q = torch.zeros((n, G, D), dtype=d64)
    q[..., :2] = torch.rand((n, G, 2), generator=g) * 3 - 1.5
    q[..., 2] = 4
    q = q.to(BF16)
    c.dq.copy_(q.repeat(B, 1, 1))
    c.dk.zero_()
    c.dv.zero_()
    rows = n * G
    p = (scale * (q.to(d64).view(rows, D)[:, :2] * 2)).exp()
    p = torch.cat((torch.ones(rows, 1, dtype=d64), p), 1)
    mine = torch.arange(D) % rows
    pd = p[mine]
    v = torch.ones((3, D), dtype=d64)
    v[1] = (-pd[:, 0] / pd[:, 1]).to(BF16).to(d64)
    v[2] = (-(pd[:, 0] + pd[:, 1] * v[1]) / pd[:, 2]).to(BF16).to(d64)
    for ids in c.slots:
        s = torch.from_numpy(ids).to(c.dk.device)
        c.dk[s[1], 0, 0], c.dk[s[2], 0, 1] = 2, 2
        c.dk[s[3:], 0, 2] = -8
        c.dv[s[:3], 0] = v.to(BF16).to(c.dv.device)
    others = torch.from_numpy(c.see[0].sum(1) - 3).repeat_interleave(G)
    total = (p.sum(1) + others * math.exp(-16))[mine]
    terms = pd * v.t()
    want, size = terms.sum(1) / total, terms.abs().sum(1) / total
    got = c.call(scale=scale).to(d64).cpu().view(B, rows, D)[:, mine, torch.arange(D)]
    worst = float((((got - want).abs() - 2.0 ** -8 * want.abs()) / size).max())
    assert worst <= 2.0 ** -20, f"2^{math.log2(worst):.2f}"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("q_lens", [[70, 3], [20, 3]])
@pytest.mark.parametrize("spread", [1.0, 40.0])
def test_infinities_under_several_operands(hip, dtype, q_lens, spread):
    """Heads of 256: an infinity in V reaches the rows that see its key, however small its
    probability, and no others; the other dims keep their bits."""
    inf = float("inf")
    c = Case(q_lens, [300, 90], 4, 2, 256, dtype, 133, 4, seed=5, spread=spread)
    keep = c.call()
    assert bool(torch.isfinite(keep).all())
    for key, x in ((2, inf), (200, -inf), (260, inf), (299, inf), (240, float("nan"))):
        d, slot = key % 256, int(c.slots[0][key])
        was = c.dv[slot, 1, d].clone()
        c.dv[slot, 1, d] = x
        got = c.call()
        c.dv[slot, 1, d] = was
        want = keep.clone()
        want[torch.from_numpy(c.see[0][:, key]).nonzero()[:, 0].to("cuda"), 2:4, d] = x
        assert torch.equal(torch.nan_to_num(got, 1e4, 2e4, 3e4), torch.nan_to_num(want, 1e4, 2e4, 3e4)), key


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n", [6, 40, 150])
@pytest.mark.parametrize("size,step", [(10, 1), (20, 8), (24, 8), (25, 4), (25, 8), (26, 8), (27, 16),
                                       (28, 32)])
@pytest.mark.parametrize("scale", [math.log(2.0), 1.0])
def test_large_scores(hip, dtype, D, n, size, step, scale):
    """Scores of 2^size and, from key 40 or 170 on, `step` more (both exact in fp32; a later one
    exceeds the first by a step of fp32 or a few): no operand overflows, and the weights are 1 and
    e^(scale step), whose exponent is off by a rounding of it and of log2(e) scale, 2^-23 of it
    each at most."""
    for turn in (40, 170):
        c = Case([n], [300], 4, 2, D, dtype, seed=size)
        c.dk.zero_()
        c.dq.zero_()
        first, second = (torch.from_numpy(s).to(c.dk.device)
                         for s in (c.slots[0][:turn], c.slots[0][turn:]))
        c.dq[:, :, 0], c.dq[:, :, 1] = 2.0 ** (size // 2), 1
        c.dk[:, :, 0] = 2.0 ** (size - size // 2)
        c.dk[second, :, 1] = step
        c.dv[first], c.dv[second] = 1.0, 0.0
        got = c.call(scale=scale).double().cpu()
        total = torch.from_numpy(c.see[0].sum(1)).double()[:, None, None]
        ones = total.clamp_max(turn)
        # of the first keys, whose value is 1
        share = ones / (ones + (total - ones) * math.exp(scale * step))
        half = torch.finfo(dtype).eps / 2
        bound = share * (2 * half * (1 + half) + 2.0 ** -21 * step + 300 * 2.0 ** -24)
        if dtype == F16:
            # the running maximum is a multiple of fp32's step at that size, up to half of one above
            # what it stands for, and the end of fp16 as much nearer
            unit = 2.0 ** (math.floor(math.log2(2.0 ** size * scale * math.log2(math.e))) - 23)
            bound = bound + 2.0 ** -25
            if D < 256:
                bound = bound + ones * 2.0 ** (-31 + unit / 2) / total
            else:
                # Three operands: the second and third are kept above 0, 2^-24 each, so a p is held
                # 2^-23 too large at most.  A row's largest p is 2^13 at first; with the running maximum
                # rounded to a step it is 2^(13 - unit / 2) to 2^(13 + unit / 2), and where that exceeds
                # 2^15 the maximum moves one step up: more than 2^(15 - unit).  The row sum, without
                # these 2^-23, is as many of the largest p as there are later keys (or all).
                largest = min(13 - unit / 2, 15 - unit)
                many = torch.where(total > ones, total - ones, total)
                bound = bound + ones * 2.0 ** (-23 - largest) / many
        err = (got - share).abs()
        assert bool(torch.isfinite(got).all()), turn
        assert bool((err <= bound).all()), (turn, float((err / bound).max()))
