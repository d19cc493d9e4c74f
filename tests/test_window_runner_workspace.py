"""A batch's workspace is allocated where a launch takes it."""

import types

import pytest
import torch

from dispec_amd.engine import model_runner
from tests.toy_lm import toy_lm


@pytest.mark.parametrize("kinds,window,max_ctx,expected", [
    (None, 0, 64, True), (None, 32, 64, False), (None, 64, 64, True), (None, 100, 64, True),
    (["sliding_attention"] * 2, 0, 64, False), (["sliding_attention", "full_attention"], 0, 64, True),
    (["sliding_attention", "full_attention"], 40, 64, False),
    (["sliding_attention"] * 2, 0, 16, True),
])
@pytest.mark.parametrize("decode", [True, False])
def test_workspace(monkeypatch, kinds, window, max_ctx, expected, decode):
    """(A window as long as the table's contexts is none: those layers run the plain launches.)"""
    model = toy_lm("qwen2")
    if kinds:
        model.config.layer_types, model.config.sliding_window = kinds, 20
    runner = model_runner.ModelRunner(model, window=window)
    made = []
    for name in ("decode_workspace", "mq_workspace"):
        monkeypatch.setattr(model_runner, name, lambda *a, name=name: made.append(name))
    monkeypatch.setattr(runner, "layers", [])
    batch = model_runner._Batch(block_table=torch.zeros(2, 4, dtype=torch.int32),
                                ctx_lens=torch.ones(2, dtype=torch.int32),
                                cu_q=torch.arange(3, dtype=torch.int32), max_q_len=1 if decode else 3,
                                max_ctx=max_ctx, decode=decode)
    cache = types.SimpleNamespace(key=torch.zeros(1))
    runner.run_batch(torch.zeros(2, dtype=torch.long), torch.zeros(2, dtype=torch.long),
                     torch.arange(2), batch, cache)
    assert made == ([("decode_workspace" if decode else "mq_workspace")] if expected else [])
