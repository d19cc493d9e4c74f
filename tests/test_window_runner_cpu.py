"""The runner's windows on the host."""

import pytest

from tests.toy_lm import toy_lm


def test_windows():
    """A runner's window and sinks, layers that have their own, and what is refused."""
    from dispec_amd.engine.model_runner import ModelRunner
    assert ModelRunner(toy_lm("qwen3")).windows == [(0, 0)] * 2
    assert ModelRunner(toy_lm("qwen3"), window=64, sinks=4).windows == [(64, 4)] * 2
    model = toy_lm("qwen2")
    model.config.layer_types = ["sliding_attention", "full_attention"]
    model.config.sliding_window = 32
    assert ModelRunner(model, window=64, sinks=4).windows == [(32, 0), (64, 4)]
    model.config.sliding_window = None
    with pytest.raises(ValueError, match="sliding_window"):
        ModelRunner(model)
    model.config.layer_types = ["chunked_attention", "full_attention"]
    with pytest.raises(ValueError, match="chunked_attention"):
        ModelRunner(model)
    for kw in (dict(window=-1), dict(sinks=4), dict(window=8, sinks=-1)):
        with pytest.raises(ValueError, match="window"):
            ModelRunner(toy_lm("qwen3"), **kw)
