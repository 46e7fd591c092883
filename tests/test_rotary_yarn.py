"""yarn's optional keys against their formulas and transformers' own rotation."""
import math

import pytest

torch = pytest.importorskip("torch")
transformers = pytest.importorskip("transformers")

YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 1024}
SMALL = dict(hidden_size=256, intermediate_size=512, num_hidden_layers=1, num_attention_heads=4, num_key_value_heads=2,
             head_dim=64, vocab_size=64, max_position_embeddings=4096)


def _theirs(scaling):
    cfg = transformers.LlamaConfig(**SMALL, rope_parameters={**scaling, "rope_theta": 10000.0})
    rope = transformers.AutoModelForCausalLM.from_config(cfg).model.rotary_emb
    return rope.inv_freq.double(), rope.attention_scaling


def _scale(m, factor):
    return 0.1 * m * math.log(factor) + 1 if factor > 1 else 1.0


@pytest.mark.parametrize("keys,mag", [
    ({}, _scale(1, 4)),
    ({"mscale": 0.7, "mscale_all_dim": 1.3}, _scale(0.7, 4) / _scale(1.3, 4)),
    ({"mscale": 1.0, "mscale_all_dim": 1.0}, 1.0),
    ({"mscale": 0.7}, _scale(1, 4)),                       # one alone says nothing
    ({"mscale_all_dim": 0.7}, _scale(1, 4)),
    ({"mscale": 1.0, "mscale_all_dim": 0.0}, _scale(1, 4)),
    ({"mscale": 0.7, "mscale_all_dim": 1.3, "attention_factor": 2.0}, 2.0),
])
def test_magnitude(keys, mag):
    from blackwell_ops.decode import rotary_frequencies

    f, got = rotary_frequencies(64, 10000.0, {**YARN, **keys})
    theirs, their_mag = _theirs({**YARN, **keys})
    assert got == pytest.approx(mag, rel=1e-14) and got == pytest.approx(their_mag, rel=1e-12)
    assert torch.allclose(theirs, f, rtol=2.0**-21, atol=0)
