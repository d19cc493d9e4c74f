"""Infinities in V reach the rows that see their keys, as infinities, on the kernels of
paged_tree_attention: whichever key a row sees first, however small the key's probability."""

import numpy as np
import pytest
import torch

from tests._tree import Case
from tests._util import f64

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
INF = float("inf")


def _check(c, got, hits, keep):
    """hits: {(row, KV head, dim): value}; the rest is `keep` and finite."""
    want = keep.clone()
    for (row, kvh, d), x in hits.items():
        want[row, kvh * c.G:(kvh + 1) * c.G, d] = x
    assert bool(torch.isfinite(keep).all())
    assert torch.equal(got, want), (got != want).nonzero()[:8].tolist()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [64, 128, 256, 32])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("n", [64, 300])
def test_a_first_key_anywhere_in_a_chunk(hip, dtype, D, sign, n):
    """Nodes that see themselves only, no context: the first key that a row sees lies anywhere."""
    c = Case([n, 3], [n, 40], 4, 2, D, dtype, seed=D, see=[np.eye(n, dtype=bool),
                                                           np.ones((3, 3), dtype=bool)])
    keep = c.call()
    hits = {}
    for i in (40, 63, 100, 170, 253, n - 1):
        if i < n:
            c.dv[int(c.slots[0][i]), i % 2, i % D] = sign * INF
            hits[(i, i % 2, i % D)] = sign * INF
    _check(c, c.call(), hits, keep)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [64, 128, 256, 32])
def test_a_first_key_behind_bad_blocks(hip, dtype, D):
    """Keys 0 to 31 have no block: the first key that counts is the chunk's 33rd."""
    c = Case([6, 2], [50, 45], 4, 2, D, dtype, seed=D + 1)
    c.bt[0, :2] = -1
    keep = c.call()
    c.dv[int(c.slots[0][33]), 1, 5] = INF
    _check(c, c.call(), {(i, 1, 5): INF for i in range(6)}, keep)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("later", [40, 100, 250])
def test_a_maximum_far_above_an_infinity(hip, dtype, D, later):
    """The key behind it scores 2^200 times as high: the infinity stays one."""
    n = 300
    see = np.zeros((n, n), dtype=bool)
    see[:, 3] = see[:, later] = True
    c = Case([n, 2], [n, 20], 4, 2, D, dtype, seed=D + 2, see=[see, np.ones((2, 2), dtype=bool)])
    c.dk[int(c.slots[0][3])] = 0
    c.dk[int(c.slots[0][later])] = 0
    c.dk[int(c.slots[0][later]), :, 0] = 200.0
    c.dq[:, :, 0] = 1.0
    keep = c.call(scale=float(np.log(2.0)))
    assert float(np.abs(f64(keep[:n]) - f64(c.v)[c.slots[0][later]].repeat(2, 0)[None]).max()) == 0
    c.dv[int(c.slots[0][3]), 0, 7] = INF
    got = c.call(scale=float(np.log(2.0)))
    _check(c, got, {(i, 0, 7): INF for i in range(n)}, keep)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [64, 128, 256, 32])
@pytest.mark.parametrize("gap", [20.0, 33.0, 60.0, 200.0])
@pytest.mark.parametrize("ctx,sink,odd", [(300, 10, 100), (300, 100, 10), (300, 297, 40),
                                          (9000, 8000, 70), (9000, 70, 8000)])
def test_an_infinity_behind_a_small_probability(hip, dtype, D, gap, ctx, sink, odd):
    """A key that every row sees, whose probability is 2^-gap of the row's largest."""
    c = Case([5, 2], [ctx, 20], 4, 2, D, dtype, seed=D + 3, see=[np.ones((5, 5), dtype=bool),
                                                               np.ones((2, 2), dtype=bool)])
    c.dk.zero_()
    c.dk[int(c.slots[0][sink]), :, 0] = gap
    c.dq[:, :, 0] = 1.0
    keep = c.call(scale=float(np.log(2.0)))
    hits = {}
    for kvh, x in ((0, INF), (1, -INF)):
        c.dv[int(c.slots[0][odd]), kvh, 3 + kvh] = x
        hits.update({(i, kvh, 3 + kvh): x for i in range(5)})
    _check(c, c.call(scale=float(np.log(2.0))), hits, keep)
