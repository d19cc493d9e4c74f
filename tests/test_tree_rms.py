"""How far paged_tree_attention is from 64 bits in the mean over a batch, which shows a lost bit that a
bound of the worst case lets pass.

A rounding to nearest is off by at most half a step, half |x|, spread evenly: by half |x| / sqrt(3) in
the root of the mean square, roundings of different numbers independent of each other.  So with o =
sum_j p_j v_j (sum_j p_j = 1), A = sum_j p_j |v_j| and

    sigma^2 = half^2 o^2                                 the output
            + half^2 sum_j (p_j v_j)^2                   where probabilities are one 16-bit operand
            + (2^-24 (sqrt(D) + sqrt(ctx) + 8) A)^2      scores and sums in fp32, a random walk of
                                                         as many steps; exponentials, weights

the mean square of err / sigma is 1/3 at most, its root 0.578; over N outputs it strays by about
1 / sqrt(N) of that.  The limit is 0.62, N 10000 and more."""

import numpy as np
import pytest
import torch

from tests._tree import Case
from tests._util import f64

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
LIMIT = 0.62
# (query heads, KV heads, head_dim, lengths of the trees, contexts)
SHAPES = [(14, 2, 64, [8, 30], [300, 900]), (8, 2, 128, [33, 1, 12], [500, 40, 1200]),
          (8, 4, 256, [20, 9], [400, 700]), (16, 4, 32, [20, 9], [400, 700]),
          (4, 4, 128, [64, 64], [70, 64])]


def one_operand(dtype, D):
    return dtype != F32 and D in (64, 128)


def attend(c, p_type=None):
    """(o, sum (p v)^2, A, ctx), each (T, Hq, D) but ctx, in 64 bits; p_type: the probabilities,
    over the row's largest, rounded to it, the sum unrounded."""
    k, v, q = f64(c.k), f64(c.v), f64(c.q)
    o, sq, A = (np.zeros(q.shape) for _ in range(3))
    ctx, at = np.zeros((len(q), 1, 1)), 0
    for b, (n, length) in enumerate(zip(c.q_lens, c.ctx)):
        seen = np.ones((n, length), dtype=bool)
        seen[:, length - n:] = c.see[b]
        ctx[at:at + n] = length
        for h in range(c.Hq):
            kk, vv = k[c.slots[b], h // c.G], v[c.slots[b], h // c.G]
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


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_mean_error(hip, dtype, shape):
    Hq, KVH, D, q_lens, ctx = shape
    c = Case(q_lens, ctx, Hq, KVH, D, dtype, seed=31)
    got = rms(c, f64(c.call()), attend(c))
    assert got <= LIMIT, got


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype,narrower", [(F32, F16), (F16, BF16), (BF16, torch.float8_e4m3fn)])
def test_the_limit_tells_a_lost_type(shape, dtype, narrower):
    """Computed here: with the probabilities' own type the error is within the limit, with the next
    narrower one (256-wide heads and the general kernel, whose probabilities are fp32: the cache's)
    it is not."""
    Hq, KVH, D, q_lens, ctx = shape
    c = Case(q_lens, ctx, Hq, KVH, D, dtype, seed=31, device="cpu")
    exact = attend(c)

    def simulated(p_type):
        return f64(torch.from_numpy(attend(c, p_type)[0]).to(dtype))

    own = dtype if one_operand(dtype, D) else F32
    assert rms(c, simulated(own), exact) <= LIMIT
    if own == F32 and dtype != F32:
        narrower = dtype
    assert rms(c, simulated(narrower), exact) > LIMIT
