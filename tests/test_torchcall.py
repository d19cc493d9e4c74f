"""The bindings that take tensors: what they leave to the Python wrappers, and that both give the same."""

import pytest
import torch

from dispec_amd import _lib
from tests._window import Case

torchcall = pytest.importorskip("dispec_amd._torchcall")


def test_every_argument_that_is_not_as_the_library_takes_it_is_left_to_the_wrapper():
    _lib.lib()
    assert _lib.torch_calls() is torchcall
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    k = torch.zeros(64, 2, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(2, 4, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    args = [q, k, None, k, None, table, None, lens, 2, 0, 0, 16, None, 1, None, None, None, None, 0]
    assert torchcall.window(*args) is None                      # CPU tensors
    for i, x in ((0, 3), (1, None), (8, "2"), (8, 1 << 80), (5, [0])):
        bad = list(args)
        bad[i] = x
        assert torchcall.window(*bad) is None
    codes, scales = torch.zeros(64, 2, 64, dtype=torch.uint8), torch.zeros(64, 2, 2, dtype=torch.uint8)
    pools = [codes, scales, codes, scales, torch.arange(2)]
    rows = torch.zeros(2, 2, 64)
    assert torchcall.append(*pools, rows, rows, None, 0) is None
    assert torchcall.gather(*pools, torch.float32, None, 0) is None
    assert torchcall.gather(*pools, "float32", None, 0) is None
    for fn, n in ((torchcall.window, 18), (torchcall.append, 8), (torchcall.gather, 9)):
        with pytest.raises(TypeError, match="arguments expected"):
            fn(*[None] * n)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [None, "fp8", "fp4"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 4)])
def test_attention_by_either_way(hip, monkeypatch, fmt, window, sinks):
    c = Case([3, 1, 40], [100, 300, 41], 4, 2, 64, torch.bfloat16, window, sinks, seed=2, fmt=fmt)
    used = []
    fast = _lib.torch_calls()

    class Watch:
        def __getattr__(self, name):
            def call(*a):
                got = getattr(fast, name)(*a)
                used.append(got is not None)
                return got
            return call

    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.empty_like(c.dq)
    monkeypatch.setattr(_lib, "torch_calls", lambda: Watch())
    a = [c.call(), c.call(err=err, out=out, scale=0.2), c.call(max_ctx=None)]
    assert used == [True] * 3 and a[1] is out
    # left to the wrapper: bounds that have to be computed, other types and layouts
    b = [c.call(max_q_len=None), c.call(q=c.dq.transpose(0, 1).contiguous().transpose(0, 1))]
    assert used[3:] == [False, True]
    c.lens = c.lens.long()
    b.append(c.call())
    assert used[5:] == [False]
    c.lens = c.lens.int()
    for x in b:
        assert torch.equal(x, a[0])
    monkeypatch.setattr(_lib, "torch_calls", lambda: None)
    assert torch.equal(c.call(), a[0]) and torch.equal(c.call(scale=0.2), out)
    monkeypatch.setattr(_lib, "torch_calls", lambda: Watch())
    with pytest.raises(ValueError, match="max_ctx"):
        c.call(max_ctx=1 << 20)
    with pytest.raises(ValueError, match="window"):
        c.call(window=-3)


@pytest.mark.gpu
def test_rows_by_either_way(hip, monkeypatch):
    from dispec_amd.kv.quant_cache import quant_append, quant_gather
    from tests._util import randn
    x = randn((2, 5, 2, 64), 1).to("cuda")
    slots = torch.tensor([3, 0, 9, 7, 1], device="cuda")
    got = []
    for way in (_lib.torch_calls, lambda: None):
        monkeypatch.setattr(_lib, "torch_calls", way)
        pools = [torch.zeros(s, dtype=torch.uint8, device="cuda")
                 for s in ((2, 16, 2, 64), (2, 16, 2, 2), (2, 16, 2, 64), (2, 16, 2, 2))]
        quant_append(*pools, slots, x, x.flip(-1))
        got.append([*pools, *quant_gather(*pools, slots, torch.float16),
                    *quant_gather(*[p[1] for p in pools], slots, torch.float32)])
        with pytest.raises(ValueError, match="slots"):
            quant_append(*pools, slots.int(), x, x)
    for a, b in zip(*got):
        assert torch.equal(a, b)
