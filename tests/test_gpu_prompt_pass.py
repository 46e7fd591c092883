"""The operators of a prompt's pass run together: the speculative decoder's packed prompts and scores, against the same
model in fp32 whose projections hold the dequantised int8 copies.

Tolerances.  A packed pass attends to 16-bit keys and values; what differs from the fp32 twin are roundings to fp16, half an
ulp at most (2^-11), 2^-11 / sqrt 3 in the mean.  A query or a key has three (the normalised row, the projection, the rotated
head): 2^-11 of itself.  With scores of spread s (sqrt of the mean fourth power of the heads' norm weights; under 1
without such norms) a score is then off by a = s sqrt 2 2^-11, and so, relatively, is a weight and what it adds to the
row; two more roundings on the way (values and output) give e1 = a + 2^-10 after the first layer.  The second layer's
queries and keys are off by that: its scores by s sqrt 2 e1, its rows by e2 = s sqrt 2 e1 + a + 2^-10 (s = 1: 0.4 %,
s = 4.4: 2.9 %).  A logit is off by e2 of the logits' spread, a log probability by its logit's error and the normaliser's,
independent of each other: sqrt 2 e2 of the spread, of which 6 standard deviations hold.  (Plain fp16 arithmetic on the same model is
as far off: 0.36 % of the last hidden state's norm over 130 tokens with s = 4.4, where the packed pass has 0.44 %.)
Steps after a packed prompt read the int8 cache: 2 % of the logits' norm (test_gpu_spec_decode)."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
transformers = pytest.importorskip("transformers")

from test_gpu_spec_decode_configs import SMALL, _pair, _rel  # noqa: E402

CONFIGS = {"qwen3": lambda: transformers.Qwen3Config(**SMALL),
           "llama": lambda: transformers.LlamaConfig(**SMALL, attention_bias=True, mlp_bias=True),
           "qwen3 128": lambda: transformers.Qwen3Config(**{**SMALL, "num_attention_heads": 8, "head_dim": 128})}


def _prompts(seed, lens, vocab=512):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, vocab, (n,), generator=g).tolist() for n in lens]


def _slack(want, mdl):
    w = [getattr(mdl.base.model.layers[0].self_attn, n, None) for n in ("q_norm", "k_norm")]
    s = 1.0 if w[0] is None else float((w[0].weight.detach().double() ** 2 * w[1].weight.detach().double() ** 2).mean().sqrt())
    a = s * 2**0.5 * 2.0**-11
    e1 = a + 2.0**-10
    e2 = s * 2**0.5 * e1 + a + 2.0**-10
    return 6 * 2**0.5 * e2 * float(want.std(-1).mean())


@torch.no_grad()
def _want(twin, prompt, dev):
    return torch.log_softmax(twin(input_ids=torch.tensor([prompt], device=dev)).logits[0, :-1].double(), -1)


@pytest.mark.parametrize("name", sorted(CONFIGS))
def test_scores(cuda_dev, name):
    from blackwell_inference.spec_decode import TreeSpeculativeDecoder

    mdl, twin = _pair(CONFIGS[name](), cuda_dev)
    with torch.no_grad():
        for layer in list(mdl.base.model.layers) + list(twin.model.layers):  # norms of the heads that matter
            for norm in (getattr(layer.self_attn, "q_norm", None), getattr(layer.self_attn, "k_norm", None)):
                if norm is not None:
                    norm.weight.copy_(torch.linspace(0.5, 3.0, norm.weight.numel()).half())
    dec = TreeSpeculativeDecoder(mdl, batch=1, max_len=700)
    prompts = _prompts(1, [130, 1, 700, 2, 0, 64, 333])
    got = dec.score(prompts, top=5, rows=300)
    assert len(got) == len(prompts) and int(dec.ctx[0]) == 0 and not bool(dec.cache.k.any())
    for s, p in zip(got, prompts):
        m = max(len(p) - 1, 0)
        assert s.logprobs.shape == s.entropy.shape == (m,) and s.top_logprobs.shape == s.top_tokens.shape == (m, 5)
        if not m:
            continue
        want = _want(twin, p, cuda_dev)
        slack = _slack(want, mdl)
        given = torch.tensor(p[1:], device=cuda_dev)
        assert float((s.logprobs - want.gather(1, given[:, None])[:, 0]).abs().max()) <= slack
        assert float((s.top_logprobs - want.topk(5).values).abs().max()) <= slack
        assert float((s.top_logprobs - want.gather(1, s.top_tokens)).abs().max()) <= slack
        entropy = -(want.exp() * want).sum(-1)
        # (dH = -sum dp (ln p + 1): at most twice the error of a log probability times the spread of ln p)
        assert float((s.entropy - entropy).abs().max()) <= 2 * slack * float(want.std(-1).max())
        alone = dec.score([p], top=5)[0]
        assert float((alone.logprobs - s.logprobs).abs().max()) <= slack
    assert dec.score([]) == [] and dec.score([[], [3]])[1].logprobs.numel() == 0


def test_scores_with_an_adapter(cuda_dev):
    from blackwell_inference.spec_decode import TreeSpeculativeDecoder

    mdl, twin = _pair(CONFIGS["qwen3"](), cuda_dev)
    g = torch.Generator(device=cuda_dev).manual_seed(7)
    mdl.load_adapter("a", {name: ((torch.randn(16, layer.in_features, generator=g, device=cuda_dev) / 16).half(),
                                  (torch.randn(layer.out_features, 16, generator=g, device=cuda_dev) * 0.05).half(), 2.0)
                           for name, layer in mdl._lora_layers.items()})
    dec = TreeSpeculativeDecoder(mdl, batch=1, max_len=100)
    prompt = _prompts(2, [80])
    plain, with_a = dec.score(prompt)[0], dec.score(prompt, adapter="a")[0]
    for name, layer in mdl._lora_layers.items():
        q, s = layer.copies["a"]
        twin.get_submodule(name).weight.data = q.float() * s.float()[:, None]
    want = _want(twin, prompt[0], cuda_dev)
    got = want.gather(1, torch.tensor(prompt[0][1:], device=cuda_dev)[:, None])[:, 0]
    slack = _slack(want, mdl)
    assert float((with_a.logprobs - got).abs().max()) <= slack < float((plain.logprobs - got).abs().max())


@pytest.mark.parametrize("name", sorted(CONFIGS))
def test_packed_prompts(cuda_dev, name):
    """Prompts of different lengths committed in one pass, then steps over the cache."""
    from blackwell_inference.spec_decode import TreeSpeculativeDecoder

    mdl, twin = _pair(CONFIGS[name](), cuda_dev)
    lens = [130, 1, 0, 517, 64]
    prompts, steps = _prompts(3, lens), torch.tensor(_prompts(4, [9] * 5), device=cuda_dev)
    for packed in (False, True):  # (either way of the steps' own norms)
        dec = TreeSpeculativeDecoder(mdl, batch=5, max_len=600, page=16, packed=packed)
        dec.prefill_packed(prompts)
        assert dec.ctx.tolist() == lens
        got = dec.forward(steps)
        for b in range(5):
            with torch.no_grad():
                want = twin(input_ids=torch.cat([torch.tensor(prompts[b], dtype=torch.int64, device=cuda_dev), steps[b]])[None])
            want = want.logits[0, lens[b]:]
            assert _rel(got[b], want) <= 2e-2, (b, _rel(got[b], want))
    # the cache holds what the prompt's keys and values are, and nothing behind them
    other = TreeSpeculativeDecoder(mdl, batch=5, max_len=600, page=16)
    other.prefill_packed(prompts)
    slot = torch.arange(other.table.shape[1] * 16, device=cuda_dev)
    for b, n in enumerate(lens):
        rows = other.cache.k[:, other.table[b].long()].movedim(2, 3).flatten(1, 2)
        assert not bool(rows[:, slot >= n].any()) and (n == 0 or bool(rows[:, slot < n].any(-1).all()))


def test_packed_decoding(cuda_dev):
    """Greedy decoding from packed prompts: each token is the model's best, or one within the logits' rounding of it."""
    from blackwell_inference.spec_decode import TreeSpeculativeDecoder
    from blackwell_ops import _lib

    mdl, twin = _pair(CONFIGS["qwen3"](), cuda_dev)
    ids = torch.tensor(_prompts(5, [40, 40], 30), device=cuda_dev).repeat(1, 3)
    dec = TreeSpeculativeDecoder(mdl, batch=2, max_len=200, nodes=12, packed=True)
    new = dec.generate(ids, 30)
    assert new.shape == (2, 30) and torch.equal(new, dec.generate(ids, 30))
    with torch.no_grad():
        logits = twin(input_ids=torch.cat([ids, new], 1)).logits[:, ids.shape[1] - 1:-1]
    best = logits.max(-1).values
    mine = logits.gather(-1, new[..., None])[..., 0]
    # two logits, each off by 2 % of the row's root mean square, 5 standard deviations
    assert bool((best - mine <= 5 * 2**0.5 * 2e-2 * logits.square().mean(-1).sqrt()).all())
    one = dec.generate(ids[:, :1], 3)  # a prompt of the root alone
    assert one.shape == (2, 3)
    assert _lib.device_status() == 0


def test_refusals(cuda_dev):
    from blackwell_inference.spec_decode import TreeSpeculativeDecoder

    mdl, _ = _pair(CONFIGS["qwen3"](), cuda_dev)
    dec = TreeSpeculativeDecoder(mdl, batch=2, max_len=20)
    for match, fn in [("at most max_len", lambda: dec.score([[1] * 21])),
                      ("at most max_len", lambda: dec.prefill_packed([[1], [1] * 21])),
                      ("each of 2 sequences", lambda: dec.prefill_packed([[1]])),
                      ("list of tokens", lambda: dec.score([[[1, 2]]])),
                      ("rows must be", lambda: dec.score([[1, 2]], rows=0)),
                      ("top must be", lambda: dec.score([[1, 2]], top=33))]:
        with pytest.raises(RuntimeError, match=match):
            fn()
