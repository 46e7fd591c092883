"""Host side of the decoder's prompts, with a model that computes nothing: no GPU."""
from types import SimpleNamespace

import pytest

torch = pytest.importorskip("torch")


class _Registry:
    """The parts of a registry that the decoder's host side reads."""

    def __init__(self, vocab):
        self.base = SimpleNamespace(model=SimpleNamespace(embed_tokens=torch.nn.Embedding(vocab, 2)))
        self.current_adapter, self.switches = None, []

    def set_adapter(self, name):
        self.current_adapter = name
        self.switches.append(name)


def _decoder(vocab=10, batch=1, max_len=8, packed=False):
    from blackwell_inference.spec_decode import TreeSpeculativeDecoder

    dec = TreeSpeculativeDecoder.__new__(TreeSpeculativeDecoder)
    dec.dev, dec.batch, dec.max_len, dec.packed, dec.nodes = torch.device("cpu"), batch, max_len, packed, 1
    dec.model = _Registry(vocab)
    dec.ctx = torch.zeros(batch, dtype=torch.int32)
    return dec


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("ids", [[[1, 2, 10]], [[1, 2, -1]], [[10]], [[-3, 2, 1]], [[1, 10, 1]]])
def test_generate_refuses_tokens_outside_the_vocabulary(ids, packed):
    """Every token, the last (the first tree's root) too: the embedding would fault on the device."""
    dec = _decoder(packed=packed)
    dec.ctx[0] = 5
    with pytest.raises(RuntimeError, match="tokens must be 0 to 9"):
        dec.generate(torch.tensor(ids), 2, adapter="a")
    assert dec.model.switches == [] and int(dec.ctx[0]) == 5  # a refused call changes nothing


def test_scores_leave_the_adapter_as_it_was(monkeypatch):
    """Steps that go on behind a score have the adapter that their sequences began with, also where the score fails."""
    import blackwell_ops.cuda
    import blackwell_ops.prompt as P

    dec = _decoder()
    dec.model.set_adapter("mine")
    dec.model.base.model.norm = SimpleNamespace(weight=None, variance_epsilon=1e-6)
    dec.model.base.lm_head = lambda x: x
    used = []

    def prompts(tokens, lens, **kw):
        used.append(dec.model.current_adapter)
        return torch.zeros((tokens.numel(), 10)), None

    monkeypatch.setattr(dec, "_prompts", prompts)
    monkeypatch.setattr(blackwell_ops.cuda, "rmsnorm", lambda x, w, eps: x)
    none = lambda logits, tokens, top: P.TokenLogprobs(*(torch.zeros((len(tokens), *shape)) for shape in ((), (), (top,), (top,))))  # noqa: E731
    monkeypatch.setattr(P, "token_logprobs", none)
    for adapter in (None, "other"):
        assert [len(s.logprobs) for s in dec.score([[1, 2, 3], [], [4]], adapter=adapter, rows=2)] == [2, 0, 0]
        assert used.pop() == adapter and dec.model.current_adapter == "mine"
        dec.score([], adapter=adapter)
        assert dec.model.current_adapter == "mine"

    def fails(*args, **kw):
        raise RuntimeError("no memory")

    monkeypatch.setattr(dec, "_prompts", fails)
    with pytest.raises(RuntimeError, match="no memory"):
        dec.score([[1, 2]], adapter="other")
    assert dec.model.current_adapter == "mine"


@pytest.mark.parametrize("packed", [False, True])
def test_generate_keeps_the_lengths_in_place(monkeypatch, packed):
    """A captured step reads the sequences' lengths where they were when it was captured."""
    import blackwell_ops.decode as D

    dec = _decoder(batch=2, max_len=20, packed=packed)
    ctx, at = dec.ctx, []

    def forward(tokens, parents=None, logits=True):
        at.append((tokens.shape[1], ctx.tolist()))
        return torch.zeros((*tokens.shape, 10)) if logits else None

    def commit(path, taken):
        dec.ctx += taken + 1

    def verify(probs, tokens, parents, u, e):  # the root's best token, and nothing drafted
        return torch.zeros(2, dtype=torch.int32), None, torch.full((2, 1), 7)

    monkeypatch.setattr(dec, "forward", forward)
    monkeypatch.setattr(dec, "commit", commit)
    monkeypatch.setattr(dec, "_prompts", lambda *a, **kw: None)
    monkeypatch.setattr(D, "verify_tree", verify)
    for n in (0, 1, 3):
        assert dec.generate(torch.tensor([[1, 2, 3], [4, 5, 6]]), n).tolist() == [[7] * n] * 2
        assert dec.ctx is ctx and ctx.tolist() == [2 + n] * 2
    assert at[-3:] == [(1, [2, 2]), (1, [3, 3]), (1, [4, 4])]


def test_prompts_go_in_passes_of_bounded_size(monkeypatch):
    """No pass has more tokens than ``pass_tokens`` but a single prompt's; every prompt is in one pass, in its own place."""
    import blackwell_ops.cuda
    import blackwell_ops.prompt as P

    lens = [3, 0, 5, 1, 0, 9, 2, 2, 4, 0]
    prompts = [[(i + 1) % 10] * n for i, n in enumerate(lens)]
    dec = _decoder(batch=len(lens), max_len=9)
    dec.model.base.model.norm = SimpleNamespace(weight=None, variance_epsilon=1e-6)
    dec.model.base.lm_head = lambda x: x
    for most in (1, 4, 8, 9, 13, 1000):
        dec.pass_tokens = most
        for write in (False, True):
            seen = [None] * len(lens)
            sizes = []

            def one(tokens, part, write=write, first=None):
                assert tokens.numel() == sum(part) and (sum(part) <= most or sum(n > 0 for n in part) == 1)
                sizes.append(sum(part))
                at = 0
                for k, n in enumerate(part):
                    if write:
                        assert seen[first + k] is None
                        seen[first + k] = tokens[at:at + n].tolist()
                    at += n
                return torch.nn.functional.one_hot(tokens, 10).float(), None

            monkeypatch.setattr(dec, "_prompts", one)
            monkeypatch.setattr(blackwell_ops.cuda, "rmsnorm", lambda x, w, eps: x)

            def logprobs(logits, tokens, top):  # the token that the row stands for
                rows = logits.argmax(-1).float() if len(logits) else torch.zeros(0)
                return P.TokenLogprobs(rows, tokens.float(), torch.zeros((len(tokens), top)), torch.zeros((len(tokens), top)))

            monkeypatch.setattr(P, "token_logprobs", logprobs)
            if write:
                dec.prefill_packed(prompts)
                assert [x or [] for x in seen] == prompts and dec.ctx.tolist() == lens
            else:
                for s, p in zip(dec.score(prompts, rows=2), prompts):
                    assert s.logprobs.tolist() == p[:-1] and s.entropy.tolist() == p[1:]
            assert sum(sizes) == sum(lens) and min(sizes) > 0
            if most == 1000:
                assert len(sizes) == 1


def test_norms_of_queries_and_keys_have_one_epsilon():
    """One launch takes both with one epsilon: layers that differ are refused, not normalised with the queries'."""
    dec = _decoder()
    norm = lambda eps: SimpleNamespace(weight=torch.ones(2), variance_epsilon=eps)  # noqa: E731
    with pytest.raises(RuntimeError, match="different epsilons"):
        dec._norms(SimpleNamespace(q_norm=norm(1e-6), k_norm=norm(1e-5)))
    assert dec._norms(SimpleNamespace(q_norm=norm(1e-5), k_norm=norm(1e-5)))["eps"] == 1e-5
    one = dec._norms(SimpleNamespace(k_norm=norm(1e-5)))
    assert one["eps"] == 1e-5 and one["q_weight"] is None
    assert dec._norms(SimpleNamespace()) == {}
