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


def _rotation(cfg, monkeypatch):
    """What the decoder asks rotary_plan for: (frequencies, magnitude)."""
    from blackwell_inference.spec_decode import TreeSpeculativeDecoder
    from blackwell_ops import decode

    asked = []

    class Reached(Exception):
        pass

    def plan(rot_dim, base=10000.0, scaling=None, interleaved=False, device=None):
        asked.append(decode.rotary_frequencies(rot_dim, base, scaling))
        raise Reached

    monkeypatch.setattr(decode, "rotary_plan", plan)
    base = types.SimpleNamespace(config=cfg, model=types.SimpleNamespace(layers=[]), parameters=lambda: iter([torch.zeros(1)]))
    with pytest.raises(Reached):
        TreeSpeculativeDecoder(types.SimpleNamespace(quantize=True, base=base), 1, 100)
    return asked[0]


LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 1024}


@pytest.mark.parametrize("scaling", [None, LLAMA3, {"type": "linear", "factor": 4.0}])
def test_configurations_that_carry_rope_scaling(scaling, monkeypatch):
    """Theta and scaling as attributes of their own, without rope_parameters."""
    from blackwell_ops.decode import rotary_frequencies

    cfg = types.SimpleNamespace(model_type="llama", hidden_size=256, num_attention_heads=4, num_key_value_heads=2,
                                hidden_act="silu", rope_theta=500000.0, rope_scaling=scaling)
    got, want = _rotation(cfg, monkeypatch), rotary_frequencies(64, 500000.0, scaling)
    assert torch.equal(got[0], want[0]) and got[1] == want[1]


@pytest.mark.parametrize("scaling", [{"rope_type": "default"}, LLAMA3, {"rope_type": "linear", "factor": 4.0},
                                     {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 1024}])
def test_rotation_of_a_configuration(scaling, monkeypatch):
    """Frequencies (fp32 in the model: 2^-21 with its powers) and magnitude of transformers' own Llama."""
    cfg = transformers.LlamaConfig(**SMALL, rope_parameters={**scaling, "rope_theta": 20000.0})
    own = transformers.AutoModelForCausalLM.from_config(cfg).model.rotary_emb
    f, mag = _rotation(cfg, monkeypatch)
    assert torch.allclose(own.inv_freq.double(), f, rtol=2.0**-21, atol=0) and own.attention_scaling == pytest.approx(mag, rel=1e-12)


@pytest.mark.parametrize("kind", ["GraniteConfig", "CohereConfig", "GemmaConfig", "SmolLM3Config"])
def test_models_with_other_layers_are_refused(kind):
    """Their modules have the same names, but embeddings or residuals are scaled, pairs interleaved, norms offset or
    layers left without positions."""
    with pytest.raises(RuntimeError, match="not supported"):
        _decoder(getattr(transformers, kind)(**SMALL, pad_token_id=0))
