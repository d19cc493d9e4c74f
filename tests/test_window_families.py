"""Which models' sliding layers the runner takes."""

import pytest

from tests.toy_lm import toy_lm


@pytest.mark.parametrize("family", ["qwen2", "qwen3"])
def test_sliding_layers_of_other_families_are_refused(family):
    """A family whose sliding layers differ from its full ones in more than the window would be
    answered wrongly; its models without sliding layers are taken as before."""
    from dispec_amd.engine.model_runner import ModelRunner
    model = toy_lm(family)
    model.config.sliding_window = 32
    model.config.layer_types = ["sliding_attention", "full_attention"]
    assert ModelRunner(model).windows == [(32, 0), (0, 0)]
    for other in ("another", None):
        model.config.model_type = other
        model.config.layer_types = ["sliding_attention", "full_attention"]
        with pytest.raises(ValueError, match="sliding-window attention layers"):
            ModelRunner(model)
        model.config.layer_types = ["full_attention"] * 2
        assert ModelRunner(model).windows == [(0, 0)] * 2
        assert ModelRunner(model, window=64, sinks=4).windows == [(64, 4)] * 2
