"""Host side of the decoding operators: no GPU."""
import pytest

torch = pytest.importorskip("torch")


def test_base_of_a_mapping():
    """A mapping's rope_theta is the base unless one is given."""
    from blackwell_ops.decode import rotary_frequencies

    mapping = {"rope_type": "linear", "factor": 2.0, "rope_theta": 500000.0}
    want = rotary_frequencies(64, 500000.0, {"rope_type": "linear", "factor": 2.0})[0]
    assert torch.equal(rotary_frequencies(64, scaling=mapping)[0], want)
    assert torch.equal(rotary_frequencies(64, 10000.0, mapping)[0], rotary_frequencies(64)[0] / 2)
    assert torch.equal(rotary_frequencies(64, scaling={"rope_type": "default"})[0], rotary_frequencies(64, 10000.0)[0])
    with pytest.raises(RuntimeError, match="base"):
        rotary_frequencies(64, scaling={"rope_theta": 0.5})


def test_without_torchs_private_calls(monkeypatch):
    """The module takes the host's shortcuts where this torch has them, and torch's public calls where it does not."""
    import importlib.util
    import sys

    from blackwell_ops import decode

    for name in ("_cuda_getCurrentRawStream", "_cuda_getDevice"):
        monkeypatch.delattr(torch._C, name, raising=False)
    monkeypatch.setitem(sys.modules, "torch._C._dynamo.guards", None)
    spec = importlib.util.spec_from_file_location("blackwell_ops.decode_bare", decode.__file__)
    bare = importlib.util.module_from_spec(spec)
    monkeypatch.setitem(sys.modules, spec.name, bare)
    spec.loader.exec_module(bare)
    assert bare._empty_strided is None
    seen = []
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda i: seen.append(i) or type("S", (), {"cuda_stream": 77}))
    assert bare._current_device() == 3 and bare._stream(3) == 77 and seen == [3]
    assert bare._new((2, 3), torch.int32, torch.device("cpu")).shape == (2, 3)
