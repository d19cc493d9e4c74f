"""Calls over quantised caches that ask for more memory than there is."""

import pytest
import torch

from dispec_amd import _lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bindings", [True, False])
def test_out_of_memory(hip, monkeypatch, bindings):
    """By either way torch's own exception, which callers catch to free something and go on."""
    from dispec_amd.kv.quant_cache import quant_gather
    if not bindings:
        monkeypatch.setattr(_lib, "torch_calls", lambda: None)
    else:
        assert _lib.torch_calls() is not None
    layers, slots = 60000, torch.zeros(1 << 16, dtype=torch.int64, device="cuda")
    codes, scales = (torch.zeros(1, 16, 2, w, dtype=torch.uint8, device="cuda").expand(layers, -1, -1, -1)
                     for w in (64, 2))
    with pytest.raises(torch.OutOfMemoryError):           # a terabyte
        quant_gather(codes, scales, codes, scales, slots)
    k, v = quant_gather(codes[0], scales[0], codes[0], scales[0], slots[:5])
    assert not k.any() and not v.any()
