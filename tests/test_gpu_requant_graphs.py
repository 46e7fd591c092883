"""Captured merge + requantisation: replays do not depend on what runs or grows outside the graph (the codes of a call
are the same each time)."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def test_graphs(cuda_dev):
    from blackwell_ops.cuda import lora_merge_requant

    g = torch.Generator(device=cuda_dev).manual_seed(1)

    def problem(n, k, r):
        return (torch.randn((n, k), generator=g, device=cuda_dev).half(), torch.randn((r, k), generator=g, device=cuda_dev).half(),
                torch.randn((n, r), generator=g, device=cuda_dev).half() * 0.02, 0.5)

    args = [problem(512, 1024, 16), problem(1000, 2048, 32)]
    junk = [torch.full((n << 20,), 0x55, dtype=torch.uint8, device=cuda_dev) for n in (1, 3)]
    del junk  # a fresh workspace does not come as zeros
    graphs, outs = [], []
    for x in args:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append([*lora_merge_requant(*x), *lora_merge_requant(*x)])
        graphs.append(gr)
    want = [lora_merge_requant(*x) for x in args]
    for i in (1, 0, 0, 1, 1):
        for y in outs[i]:
            y.zero_()
        graphs[i].replay()
        torch.cuda.synchronize(cuda_dev)
        for y, w in zip(outs[i], want[i] * 2):
            assert torch.equal(y, w)
    from blackwell_ops import _lib

    assert _lib.device_status() == 0
