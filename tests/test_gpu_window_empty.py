"""Windowed and quantised attention of batches in which no sequence has a token."""

import pytest
import torch

from dispec_amd.engine.hip_attn import paged_quant_attention, paged_window_attention

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("B", [1, 3000])
@pytest.mark.parametrize("D,dtype,quant", [(64, torch.bfloat16, False), (128, torch.float16, True),
                                           (64, torch.float32, True), (64, torch.float32, False),
                                           (32, torch.bfloat16, False)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3)])
@pytest.mark.parametrize("max_ctx", [0, 1, None])
def test_no_tokens(hip, B, D, dtype, quant, window, sinks, max_ctx):
    """One query a sequence without a context (a decode that is padded): zeros."""
    q = torch.randn(B, 4, D, device=DEV).to(dtype)
    table = torch.full((B, 1), -1, dtype=torch.int32, device=DEV)
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    kw = dict(window=window, sinks=sinks, max_ctx=max_ctx, err=err)
    if quant:
        codes = torch.zeros(32, 2, D, dtype=torch.uint8, device=DEV)
        scales = torch.zeros(32, 2, D // 32, dtype=torch.uint8, device=DEV)
        got = paged_quant_attention(q, codes, scales, codes, scales, table, None, lens, 2, **kw)
    else:
        rows = torch.full((32, 2, D), float("nan"), device=DEV).to(dtype)
        got = paged_window_attention(q, rows, rows, table, None, lens, 2, **kw)
    assert not got.any() and not int(err)
