"""Which configurations the speculative decoder takes: what it cannot compute as the model does, it refuses."""
import types

import pytest

torch = pytest.importorskip("torch")
transformers = pytest.importorskip("transformers")

SMALL = dict(hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
             head_dim=64, vocab_size=512, max_position_embeddings=4096)


def _decoder(cfg, max_len=100, nodes=16):
    """The constructor up to its first tensor: a model on no device stands in for the registry's."""
    from blackwell_inference.spec_decode import TreeSpeculativeDecoder

    class Reached(Exception):
        pass

    class Base:
        config = cfg
        model = types.SimpleNamespace(layers=[])

        def parameters(self):
            raise Reached

    try:
        TreeSpeculativeDecoder(types.SimpleNamespace(quantize=True, base=Base()), 1, max_len, nodes)
    except Reached:
        return True


def test_plain_configurations_are_taken():
    assert _decoder(transformers.Qwen3Config(**SMALL)) and _decoder(transformers.LlamaConfig(**SMALL))
    assert _decoder(transformers.Qwen2Config(**SMALL)) and _decoder(transformers.MistralConfig(**SMALL))


@pytest.mark.parametrize("cfg", [
    lambda: transformers.MistralConfig(**SMALL, sliding_window=64),
    lambda: transformers.Qwen3Config(**SMALL, use_sliding_window=True, sliding_window=64, max_window_layers=1),
    lambda: transformers.Qwen2Config(**SMALL, use_sliding_window=True, sliding_window=64, max_window_layers=1),
])
def test_windows_shorter_than_the_text_are_refused(cfg):
    with pytest.raises(RuntimeError, match="window"):
        _decoder(cfg(), max_len=100)
    with pytest.raises(RuntimeError, match="window"):
        _decoder(cfg(), max_len=49)  # the last tree's nodes would lie past it
    assert _decoder(cfg(), max_len=48)


def test_other_kinds_of_attention_are_refused():
    cfg = transformers.Qwen3Config(**SMALL)
    cfg.layer_types = ["full_attention", "chunked_attention"]
    with pytest.raises(RuntimeError, match="chunked_attention"):
        _decoder(cfg)


def test_partial_rotation_is_refused():
    cfg = transformers.LlamaConfig(**SMALL)
    cfg.rope_parameters = {"rope_type": "default", "rope_theta": 1e4, "partial_rotary_factor": 0.5}
    with pytest.raises(RuntimeError, match="partial_rotary_factor"):
        _decoder(cfg)
    cfg.rope_parameters = {"rope_type": "default", "rope_theta": 1e4, "partial_rotary_factor": 1.0}
    assert _decoder(cfg)
    cfg.partial_rotary_factor = 0.25  # where older configurations keep it
    with pytest.raises(RuntimeError, match="partial_rotary_factor"):
        _decoder(cfg)
