"""The speculative decoder on configurations that leave the plain Qwen3 path: logits against the same model in fp32 whose
projections hold the dequantised int8 copies.

Two layers with an int8 cache and fp16 activations: a code is off by up to half a step, uniformly, a step being a 127th of
a head row's maximum (under 3 standard deviations of 64 normals): 3 / 127 / sqrt 12 = 0.7 % of a row, in k and in v,
averaged over the keys a row sees; with fp16's roundings (2^-11 a step, some ten steps a layer) under 2 % of the logits'
norm.  What a test is after changes the logits by far more."""
import copy

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
transformers = pytest.importorskip("transformers")

SMALL = dict(hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
             head_dim=64, vocab_size=512, max_position_embeddings=4096)


def _pair(cfg, dev, seed=0, **registry):
    """(registry, fp32 twin): random weights, biases where the model has them."""
    from blackwell_inference.lora import MultiDeltaLoRAModel
    from blackwell_inference.lora.delta_multi import W8A16Linear

    torch.manual_seed(seed)
    model = transformers.AutoModelForCausalLM.from_config(cfg).to(dev, torch.float16).eval()
    with torch.no_grad():
        for m in model.modules():
            if isinstance(m, torch.nn.Linear) and m.bias is not None:
                m.bias.normal_(0, 0.5)
    twin = copy.deepcopy(model).float()
    mdl = MultiDeltaLoRAModel(model, device=str(dev), **registry)
    for name, layer in mdl._lora_layers.items():
        assert isinstance(layer, W8A16Linear)
        q, s = layer.copies[None]
        twin.get_submodule(name).weight.data = q.float() * s.float()[:, None]
    return mdl, twin


def _rel(a, b):
    return float((a.float() - b.float()).norm() / b.float().norm())


def _logits(mdl, ids, prefill=30, max_len=None):
    from blackwell_inference.spec_decode import TreeSpeculativeDecoder

    dec = TreeSpeculativeDecoder(mdl, batch=ids.shape[0], max_len=max_len or ids.shape[1] + 8, page=16)
    dec.prefill(ids[:, :prefill])
    return dec.forward(ids[:, prefill:])


def _ids(dev, n=40, vocab=512):
    return torch.randint(0, vocab, (2, n), generator=torch.Generator().manual_seed(1)).to(dev)


@torch.no_grad()
def _check(cfg, dev, **registry):
    mdl, twin = _pair(cfg, dev, **registry)
    ids = _ids(dev)
    want = twin(input_ids=ids).logits[:, 30:]
    got = _logits(mdl, ids)
    assert got.shape == want.shape and _rel(got, want) <= 2e-2, _rel(got, want)
    return mdl, twin, ids, want


def test_mlp_and_attention_biases(cuda_dev):
    mdl, twin, ids, want = _check(transformers.LlamaConfig(**SMALL, mlp_bias=True, attention_bias=True), cuda_dev)
    for layer in twin.model.layers:
        layer.mlp.gate_proj.bias = layer.mlp.up_proj.bias = layer.mlp.down_proj.bias = None
    with torch.no_grad():
        assert _rel(twin(input_ids=ids).logits[:, 30:], want) > 0.1  # the biases matter


@pytest.mark.parametrize("act", ["gelu", "relu"])
def test_other_activations(cuda_dev, act):
    mdl, twin, ids, want = _check(transformers.LlamaConfig(**SMALL, hidden_act=act), cuda_dev)
    for layer in twin.model.layers:
        layer.mlp.act_fn = torch.nn.SiLU()
    with torch.no_grad():
        assert _rel(twin(input_ids=ids).logits[:, 30:], want) > 0.05  # the activation matters


@pytest.mark.parametrize("targets", [("q_proj", "k_proj", "v_proj", "o_proj"), ("q_proj", "up_proj")])
def test_registry_of_some_projections(cuda_dev, targets):
    """The projections that the registry does not hold stay the model's own fp16 linears."""
    _check(transformers.Qwen3Config(**SMALL), cuda_dev, targets=targets)


def test_window_longer_than_the_text(cuda_dev):
    """A window that no token of max_len leaves changes nothing."""
    _check(transformers.MistralConfig(**SMALL, sliding_window=64), cuda_dev)


def test_qwen2(cuda_dev):
    """Biases of q, k and v alone, no norms of the heads."""
    _check(transformers.Qwen2Config(**SMALL), cuda_dev)


def test_no_new_tokens(cuda_dev):
    from blackwell_inference.spec_decode import TreeSpeculativeDecoder

    mdl, _ = _pair(transformers.Qwen3Config(**SMALL), cuda_dev)
    dec = TreeSpeculativeDecoder(mdl, batch=2, max_len=50)
    new = dec.generate(_ids(cuda_dev), 0)
    assert new.shape == (2, 0) and new.dtype == dec.generate(_ids(cuda_dev), 1).dtype == torch.int64
    with pytest.raises(RuntimeError, match="max_new_tokens"):
        dec.generate(_ids(cuda_dev), -1)
    with pytest.raises(RuntimeError, match="max_len"):
        dec.generate(_ids(cuda_dev), 11)
    with pytest.raises(RuntimeError, match="ids must be"):
        dec.generate(_ids(cuda_dev)[:1], 1)
