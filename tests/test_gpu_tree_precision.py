"""How many bits paged_tree_attention keeps of its probabilities, and what they depend on."""

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
