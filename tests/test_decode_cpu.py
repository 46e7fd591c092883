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
