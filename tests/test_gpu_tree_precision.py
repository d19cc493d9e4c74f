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
