"""The published ctypes bindings: their workspaces, with the library and the GPUs played by the test."""
import contextlib
import os
import re
import types
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

ROOT = Path(__file__).resolve().parent.parent
BLOCKS = re.findall(r"```python\n(.*?)```", (ROOT / "INTEGRATION.md").read_text(), re.S)


class Library:
    """Every entry point succeeds and is recorded; a workspace of `need` bytes."""

    def __init__(self, need):
        self.need, self.capture, self.calls = need, 0, []

    def __getattr__(self, name):
        def call(*args):
            if name.endswith("_workspace_size"):
                return self.need
            if name == "bw_stream_capture_id":
                args[1]._obj.value = self.capture
                return 0
            self.calls.append((name, args))
            return 0

        return call


def _tensor(shape, device, dtype=torch.float16):
    stride = [1]
    for n in shape[:0:-1]:
        stride.insert(0, stride[0] * n)
    return types.SimpleNamespace(shape=shape, device=device, dtype=dtype, data_ptr=lambda: 64, is_cuda=True,
                                 stride=lambda i=None: tuple(stride) if i is None else stride[i])


@pytest.fixture
def binding(monkeypatch):
    from blackwell_ops import _lib

    monkeypatch.setitem(os.environ, "BW_OPS_LIB", str(_lib.LIB_PATH))
    ns = {}
    for block in BLOCKS:
        if any(f"def {name}(" in block for name in ("lora_delta", "int8_gemm", "int8_gemm_swiglu", "tree_attention")):
            exec(block, ns)
    current = []
    zeros, empty = torch.zeros, torch.empty
    monkeypatch.setattr(torch, "zeros", lambda *a, device=None, **k: zeros(*a, **k))
    monkeypatch.setattr(torch, "empty", lambda *a, device=None, **k: empty(*a, **k))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device: types.SimpleNamespace(cuda_stream=0))

    @contextlib.contextmanager
    def on(device):
        current.append(device)
        yield
        current.pop()

    monkeypatch.setattr(torch.cuda, "device", on)
    ns["current"] = current
    return ns


def _call(ns, op, device, library):
    """The workspace's address in one call of `op` on `device`, whose streams all have the handle 0."""
    ns["_bw"] = library
    t = lambda *shape, dtype=torch.float16: _tensor(shape, device, dtype)  # noqa: E731
    seen = []
    entry = {"tree_attention": "bw_tree_attention_int8", "int8_gemm": "bw_w8a16_gemm",
             "int8_gemm_swiglu": "bw_w8a16_gemm_swiglu"}[op]
    record = lambda *args: seen.append((args[-3], list(ns["current"]))) or 0  # noqa: E731
    setattr(library, entry, record)
    if op == "tree_attention":
        ns[op](t(1, 2, 4, 64), t(3, 2, 16, 64), *(t(3, 2, 16) for _ in range(3)), t(1, 3), t(1), None)
    elif op == "int8_gemm":
        ns[op](t(4, 64), t(32, 64, dtype=torch.int8), t(32))
    else:
        ns[op](t(4, 64), t(32, 64), t(32), t(32, 64), t(32))
    (ws, on), = seen
    assert on == [device], "the call does not run on its tensors' device"
    return ws


@pytest.mark.parametrize("op", ["tree_attention", "int8_gemm", "int8_gemm_swiglu"])
def test_workspaces(binding, op):
    one, two = torch.device("cuda", 0), torch.device("cuda", 1)
    lib = Library(8192)
    first = _call(binding, op, one, lib)
    assert first and first == _call(binding, op, one, lib)
    assert first != _call(binding, op, two, lib), "two devices' default streams share a workspace"
    lib.capture = 5
    captured = _call(binding, op, one, lib)
    assert captured != first, "a graph shares the workspace of the calls outside"
    lib.need = 1 << 20
    assert _call(binding, op, one, lib) != captured
    assert any(w.data_ptr() == captured for kept in binding["_ws"].values() for w in kept), "a graph's workspace was freed"
    lib.need, lib.capture = 8192, 6
    assert _call(binding, op, one, lib) != captured
    lib.capture = 0
    assert _call(binding, op, one, lib) == first
    lib.need = 0
    assert _call(binding, op, one, lib) is None
