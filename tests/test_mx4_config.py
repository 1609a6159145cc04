"""The options that keep weights and activations in 4 bits, on the host."""
import pytest

from cuca_b200.config.engine_config import EngineConfigError, LocalModelConfig


def test_options():
    assert LocalModelConfig.from_json({"source": "x"}).weight_dtype is None
    config = LocalModelConfig.from_json({"source": "x", "weight_dtype": "mxfp4", "activation_dtype": "mxfp4"})
    config.validate()
    for bad in ({"weight_dtype": "int4"}, {"weight_dtype": "mxfp4", "activation_dtype": "int8"}, {"activation_dtype": "mxfp4"}):
        with pytest.raises(EngineConfigError):
            LocalModelConfig.from_json({"source": "x", **bad}).validate()


def test_models_whose_layers_do_not_take_weights_in_4_bits_are_refused():
    import pafutar_util
    import tiny
    from cuca_b200.config.registry import build_spec
    from cuca_b200.models.model import Model
    Model(build_spec(tiny.CONFIGS["B"])).check_small_weights()
    with pytest.raises(ValueError, match="4 bits"):
        Model(build_spec(pafutar_util.CONFIGS["wide"])).check_small_weights()
