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
