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


@pytest.mark.parametrize("betas", [{}, {"beta_fast": 20.0, "beta_slow": 3.0}])
def test_ends_of_the_ramp(betas):
    """truncate False: the ramp runs between the fractional pairs that turn beta_fast and beta_slow times."""
    from blackwell_ops.decode import rotary_frequencies

    keys = {**YARN, **betas, "truncate": False}
    f, _ = rotary_frequencies(64, 10000.0, keys)
    plain = 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    at = [64 * math.log(1024 / (betas.get(k, d) * 2 * math.pi)) / (2 * math.log(10000.0)) for k, d in (("beta_fast", 32.0), ("beta_slow", 1.0))]
    ramp = ((torch.arange(32, dtype=torch.float64) - at[0]) / (at[1] - at[0])).clamp(0, 1)
    assert torch.allclose(f, plain * (1 - ramp) + plain / 4 * ramp, rtol=1e-12, atol=0)
    assert torch.allclose(_theirs(keys)[0], f, rtol=2.0**-20, atol=0)
    whole, _ = rotary_frequencies(64, 10000.0, {**keys, "truncate": True})
    assert torch.equal(whole, rotary_frequencies(64, 10000.0, {**YARN, **betas})[0]) and not torch.equal(whole, f)
