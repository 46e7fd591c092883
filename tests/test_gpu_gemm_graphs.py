"""Captured W8A16 GEMM calls whose split tiles meet in the workspace: replays do not depend on what runs or grows
outside the graph.  A call's summation order is fixed, so every comparison is exact."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def _inputs(dev, m, n, k, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn((m, k), generator=g, device=dev).half(),
            torch.randint(-127, 128, (n, k), generator=g, device=dev, dtype=torch.int8),
            (torch.rand(n, generator=g, device=dev) * 1e-3 + 1e-4).half())


def _need(m, n, k):
    from blackwell_ops._lib import lib

    return lib.bw_w8a16_gemm_workspace_size(m, n, k)


def test_graphs(cuda_dev):
    """Two graphs on torch's capture stream without a warm-up, the later one replayed first; a larger eager call and
    other tensors after the captures."""
    from blackwell_ops.kernels import int8_gemm

    shapes = [(16, 1024, 4096), (8, 2048, 8192)]
    big = (128, 4096, 8192)
    assert all(_need(*s) > 0 for s in shapes) and _need(*big) > max(_need(*s) for s in shapes)
    args = [_inputs(cuda_dev, *s, i) for i, s in enumerate(shapes)]
    junk = [torch.full((n << 20,), 0x55, dtype=torch.uint8, device=cuda_dev) for n in (1, 3, 12)]
    del junk  # a fresh workspace does not come as zeros
    graphs, outs = [], []
    st = torch.cuda.Stream(cuda_dev)
    for x in args:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs.append([int8_gemm(*x), int8_gemm(*x)])
        graphs.append(g)
    with torch.cuda.stream(st):
        int8_gemm(*_inputs(cuda_dev, *big, 9))
        others = [torch.full((n << 20,), 0x55, dtype=torch.uint8, device=cuda_dev) for n in (1, 2, 4, 8)]
    torch.cuda.synchronize(cuda_dev)
    want = [int8_gemm(*x) for x in args]
    for i in (1, 0, 0, 1):
        for y in outs[i]:
            y.zero_()
        graphs[i].replay()
        torch.cuda.synchronize(cuda_dev)
        assert all(torch.equal(y, want[i]) for y in outs[i])
    assert all(bool((x == 0x55).all()) for x in others)
    ref = args[0][0].float() @ (args[0][1].float() * args[0][2].float()[:, None]).T
    assert float((want[0].float() - ref).norm() / ref.norm()) <= 2.0**-11
