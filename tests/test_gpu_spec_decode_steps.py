"""Speculation saves steps and leaves the distribution alone: models whose next token is known by construction."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
transformers = pytest.importorskip("transformers")


def _successor_model(dev, vocab, sharp):
    """Attention and MLP add nothing, so the logits after token x are sharp * cos(head row, embedding of x), and token
    x + 1's head row is x's embedding: x + 1 scores sharp, the others a random fraction of it."""
    from blackwell_inference.lora import MultiDeltaLoRAModel

    cfg = transformers.Qwen3Config(hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                                   num_key_value_heads=2, head_dim=64, vocab_size=vocab, tie_word_embeddings=False)
    torch.manual_seed(0)
    model = transformers.AutoModelForCausalLM.from_config(cfg).to(dev, torch.float16).eval()
    with torch.no_grad():
        for layer in model.model.layers:
            layer.self_attn.o_proj.weight.zero_()
            layer.mlp.down_proj.weight.zero_()
        e = torch.nn.functional.normalize(torch.randn((vocab, 256), device=dev), dim=-1)
        model.model.embed_tokens.weight.copy_(e)
        model.lm_head.weight.copy_(e.roll(1, 0) * (sharp / 16))  # (the norm scales an embedding to 256 ** 0.5)
    return MultiDeltaLoRAModel(model, device=str(dev))


def test_accepted_drafts_save_steps(cuda_dev):
    """A certain cycle, seen three times in the prompt: every draft is right, so a step gives the root's token and three
    drafted ones (eleven drafts in four branches, which here are one)."""
    from blackwell_inference.spec_decode import TreeSpeculativeDecoder

    mdl = _successor_model(cuda_dev, 8, 100.0)
    ids = torch.arange(24, device=cuda_dev)[None].repeat(2, 1) % 8
    ids[1] = (ids[1] + 3) % 8
    steps = {}
    for nodes in (1, 12):
        dec = TreeSpeculativeDecoder(mdl, batch=2, max_len=80, nodes=nodes)
        calls, forward = [], dec.forward

        def counted(tokens, parents=None, logits=True):
            calls.append(logits)
            return forward(tokens, parents, logits)

        dec.forward = counted
        for temperature in (0.0, 1.0):
            calls.clear()
            new = dec.generate(ids, 40, temperature=temperature, generator=torch.Generator(cuda_dev).manual_seed(1))
            assert torch.equal(new, (ids[:, -1:] + 1 + torch.arange(40, device=cuda_dev)) % 8)
            steps[nodes, temperature] = sum(calls)
    assert steps[1, 0.0] == steps[1, 1.0] == 40
    # 4 tokens a step until fewer than 12 are left, when the trees shrink
    assert steps[12, 0.0] == steps[12, 1.0] <= 14


def test_sampled_tokens_are_the_models(cuda_dev):
    """The first sampled token of 4000 prompts, drafted or not, against the model's own probabilities: each of 12
    frequencies within 5 standard deviations."""
    from blackwell_inference.spec_decode import TreeSpeculativeDecoder

    mdl = _successor_model(cuda_dev, 12, 2.0)
    ids = (torch.arange(36, device=cuda_dev) % 12)[None].repeat(400, 1)
    dec = TreeSpeculativeDecoder(mdl, batch=400, max_len=48, nodes=4)
    dec.prefill(ids[:, :-1])
    p = torch.softmax(dec.forward(ids[:, -1:])[0, 0].double(), -1)
    assert 0.2 < float(p[0]) < 0.8  # neither certain nor hopeless: drafts are accepted and rejected
    g = torch.Generator(cuda_dev).manual_seed(2)
    for new in (2, 4):  # (with one token to go there is no draft)
        first = torch.cat([dec.generate(ids, new, temperature=1.0, generator=g)[:, 0] for _ in range(10)])
        freq = torch.bincount(first, minlength=12).double() / first.numel()
        sd = (p * (1 - p) / first.numel()).sqrt()
        assert bool(((freq - p).abs() <= 5 * sd).all()), ((freq - p) / sd).tolist()
