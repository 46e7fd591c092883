"""The speculative decoder over the registry: a Qwen3-style model (Qwen3-0.6B layer shapes, 2 layers, random init).

Logits are compared with the same model in fp32 whose projections hold the dequantised int8 copies.  What differs is the
int8 cache and fp16 activations: a code is off by up to half a step, uniformly, a step being a 127th of a head row's
maximum (about 3 standard deviations of 128 normals): 3 / 127 / sqrt 12 = 0.7 % of a row, in k and in v, averaged over
the keys a row sees; with fp16's roundings (2^-11 a step, some ten steps a layer) under 2 % of the logits' norm for two
layers.
"""
import copy

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
transformers = pytest.importorskip("transformers")


@pytest.fixture(scope="module")
def setup(cuda_dev):
    from blackwell_inference.lora import MultiDeltaLoRAModel
    from transformers import AutoModelForCausalLM, Qwen3Config

    cfg = Qwen3Config(hidden_size=1024, intermediate_size=3072, num_hidden_layers=2, num_attention_heads=16,
                      num_key_value_heads=8, head_dim=128, vocab_size=4096, tie_word_embeddings=True,
                      max_position_embeddings=4096)
    torch.manual_seed(0)
    model = AutoModelForCausalLM.from_config(cfg).to(cuda_dev, torch.float16).eval()
    plain = copy.deepcopy(model)
    mdl = MultiDeltaLoRAModel(model, device=str(cuda_dev))
    g = torch.Generator(device=cuda_dev).manual_seed(7)
    adapter = {}
    for name, layer in mdl._lora_layers.items():
        n, k = layer.out_features, layer.in_features
        adapter[name] = ((torch.randn(16, k, generator=g, device=cuda_dev) / k ** 0.5).half(),
                         (torch.randn(n, 16, generator=g, device=cuda_dev) * 0.02).half(), 2.0)
    mdl.load_adapter("a", adapter)
    return plain, mdl


def _twin(plain, mdl, adapter):
    twin = copy.deepcopy(plain).float()
    for name, layer in mdl._lora_layers.items():
        q, s = layer.copies[adapter]
        parent, _, attr = name.rpartition(".")
        lin = torch.nn.Linear(layer.in_features, layer.out_features, bias=False, device=q.device)
        lin.weight.data = q.float() * s.float()[:, None]
        setattr(twin.get_submodule(parent), attr, lin)
    return twin


def _rel(a, b):
    return float((a.float() - b.float()).norm() / b.float().norm())


@pytest.mark.parametrize("adapter", [None, "a"])
def test_chain_logits(setup, cuda_dev, adapter):
    from blackwell_inference.spec_decode import TreeSpeculativeDecoder

    plain, mdl = setup
    ids = torch.randint(0, 4096, (2, 150), generator=torch.Generator().manual_seed(1)).to(cuda_dev)
    mdl.set_adapter(adapter)
    dec = TreeSpeculativeDecoder(mdl, batch=2, max_len=200, page=16)
    dec.prefill(ids[:, :129])
    got = dec.forward(ids[:, 129:])
    with torch.no_grad():
        want = _twin(plain, mdl, adapter)(input_ids=ids).logits[:, 129:]
    assert got.shape == want.shape and _rel(got, want) <= 2e-2, _rel(got, want)


def test_tree_logits_and_commit(setup, cuda_dev):
    """Each node's logits are those of the chain of its ancestors, before and after a path is committed."""
    from blackwell_inference.spec_decode import TreeSpeculativeDecoder

    plain, mdl = setup
    g = torch.Generator().manual_seed(2)
    ids = torch.randint(0, 4096, (2, 40), generator=g).to(cuda_dev)
    tree = torch.randint(0, 4096, (2, 9), generator=g).to(cuda_dev)
    par = [[-1, 0, 0, 1, 1, 2, 4, 4, 7], [-1, 0, 1, 2, 3, 0, 5, 6, -1]]
    mdl.set_adapter(None)
    dec = TreeSpeculativeDecoder(mdl, batch=2, max_len=80, nodes=9, page=16)
    dec.prefill(ids)
    parents = torch.tensor(par, dtype=torch.int32, device=cuda_dev)
    got = dec.forward(tree, parents)
    twin = _twin(plain, mdl, None)

    def chain(b, node):
        c = []
        while node >= 0:
            c.append(node)
            node = par[b][node]
        return c[::-1]

    with torch.no_grad():
        for b in range(2):
            for node in range(9):
                if node and par[b][node] < 0:
                    continue
                c = chain(b, node)
                want = twin(input_ids=torch.cat([ids[b], tree[b, c]])[None]).logits[0, -1]
                assert _rel(got[b, node], want) <= 2e-2, (b, node, _rel(got[b, node], want))
        paths = [[1, 4, 7, 8], [5, 6, 7]]
        path = torch.tensor([p + [-1] * (9 - len(p)) for p in paths], dtype=torch.int32, device=cuda_dev)
        dec.commit(path, torch.tensor([4, 3], dtype=torch.int32, device=cuda_dev))
        assert dec.ctx.tolist() == [45, 44]
        nxt = torch.tensor([[5], [6]], device=cuda_dev)
        got = dec.forward(nxt)
        for b in range(2):
            want = twin(input_ids=torch.cat([ids[b], tree[b, [0] + paths[b]], nxt[b]])[None]).logits[0, -1]
            assert _rel(got[b, 0], want) <= 2e-2


def test_generate(setup, cuda_dev):
    """Greedy decoding by trees gives, position by position, the plain decoder's best token (or one whose logit is
    within its own rounding of the best), and repeats itself; drafts are accepted on a repetitive prompt."""
    from blackwell_inference.spec_decode import TreeSpeculativeDecoder

    _, mdl = setup
    ids = torch.randint(0, 50, (2, 48), generator=torch.Generator().manual_seed(3)).repeat(1, 2).to(cuda_dev)
    dec = TreeSpeculativeDecoder(mdl, batch=2, max_len=200, nodes=12)
    steps = 0
    forward = dec.forward

    def counted(*a, **k):
        nonlocal steps
        steps += 1
        return forward(*a, **k)

    dec.forward = counted
    new = dec.generate(ids, 40, adapter="a")
    assert new.shape == (2, 40) and torch.equal(new, dec.generate(ids, 40, adapter="a"))
    one = TreeSpeculativeDecoder(mdl, batch=2, max_len=200, nodes=1)
    one.reset()
    seq = torch.cat([ids, new], 1)
    one.prefill(seq[:, :ids.shape[1] - 1])
    for i in range(40):
        at = ids.shape[1] - 1 + i
        logits = one.forward(seq[:, at:at + 1])[:, 0].float()
        one.ctx += 1
        best = logits.max(-1).values
        mine = logits.gather(1, new[:, i:i + 1])[:, 0]
        assert bool((best - mine <= 2e-2 * logits.norm(dim=-1) / np.sqrt(logits.shape[-1])).all()), i
    # sampling: reproducible from the generator, and the drafts do not change the first token's choice set
    a = dec.generate(ids, 8, temperature=1.0, generator=torch.Generator(cuda_dev).manual_seed(5))
    b = dec.generate(ids, 8, temperature=1.0, generator=torch.Generator(cuda_dev).manual_seed(5))
    assert torch.equal(a, b) and int(a.min()) >= 0 and int(a.max()) < 4096
    from blackwell_ops import _lib

    assert _lib.device_status() == 0
