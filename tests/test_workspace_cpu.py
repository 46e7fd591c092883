"""Which scratch memory a call gets, eagerly and inside stream captures, with the stream and its capture played by the
test: a CUDA graph keeps the addresses of its capture, so no other call may be given them, or give them back."""
import weakref

import pytest

torch = pytest.importorskip("torch")

DEV = torch.device("cpu", 0)


class Stream:
    handle, capture = 7, 0  # of the class: one stream at a time


def _attention(n):
    from blackwell_ops import decode

    return decode._workspace(DEV, n)


def _gemm(n):
    from blackwell_ops.kernels import int8_gemm as _  # noqa: F401  (the operator; its module holds the workspaces)
    import sys

    return sys.modules["blackwell_ops.kernels.int8_gemm"]._workspace(DEV, Stream.handle, n)


def _requant(n):
    from blackwell_ops import cuda

    return cuda._workspace(DEV, n)


@pytest.fixture
def stream(monkeypatch):
    from blackwell_ops import _lib, cuda, decode

    s = Stream
    s.handle, s.capture = 7, 0

    def info(handle, out):
        out._obj.value = s.capture
        return 0

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: s.capture != 0)
    monkeypatch.setattr(_lib.lib, "bw_stream_capture_id", info, raising=False)
    monkeypatch.setattr(decode, "_stream", lambda index: s.handle)
    monkeypatch.setattr(cuda, "stream_ptr", lambda dev: s.handle)
    yield s


@pytest.mark.parametrize("get", [_attention, _gemm, _requant])
def test_a_capture_has_its_own(stream, get):
    eager = get(3 << 20)
    assert not eager.any() and get(1 << 20) is eager
    stream.capture = 41
    first = get(2 << 20)
    assert first is not eager, "a graph would share its tickets with the calls outside"
    assert get(1 << 20) is first, "one workspace, cleared once, for a capture"
    stream.handle = 8  # a second stream of the same capture runs beside the first
    beside = get(2 << 20)
    assert beside is not first
    stream.handle, stream.capture = 7, 42
    second = get(2 << 20)
    assert second is not first, "two graphs would share a workspace, cleared by the first alone"
    stream.capture = 0
    assert get(2 << 20) is eager


@pytest.mark.parametrize("get", [_attention, _gemm, _requant])
def test_growth_leaves_a_graphs_memory_alone(stream, get):
    stream.capture = 51
    held = weakref.ref(get(2 << 20))
    stream.capture = 0
    big = get(20 << 20)
    assert held() is not None and held().data_ptr() != big.data_ptr()
    assert big.numel() >= 20 << 20 and not big.any()


@pytest.mark.parametrize("get,zeroed", [(_attention, 4096), (_gemm, 4096), (_requant, None)])
def test_what_a_capture_clears(stream, get, zeroed, monkeypatch):
    """The words that have to be zero are cleared by the capture itself (so by each replay); None: all of them."""
    stream.capture = 61
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, **k: empty(*a, **k).fill_(7))
    ws = get(2 << 20)
    assert not ws[:zeroed].any() and (zeroed is None or bool((ws[zeroed:] == 7).all()))


def test_capture_id_refusal():
    from blackwell_ops import _lib

    assert _lib.lib.bw_stream_capture_id(None, None) == _lib.BW_ERR_INVALID_ARGUMENT
