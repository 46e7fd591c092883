"""The same call gives the same bits every time, also started on an idle GPU, when weights come from L2 the fastest (a
weight slot given back while its rows were still being read changed some rows of fp16 tiles in one of 150 to 500 calls)."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("glu", [True, False])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(256, 4096, 2048), (130, 2560, 1024), (64, 4096, 2048), (16, 4096, 2048)])
def test_repeated_calls(cuda_dev, m, n, k, dt, glu):
    """Eight weights in turn, so that what lies in shared memory is another call's."""
    from blackwell_ops.kernels import int8_gemm, int8_gemm_swiglu

    g = torch.Generator(device=cuda_dev).manual_seed(m + n)
    calls = []
    for _ in range(8):
        x = torch.randn((m, k), generator=g, device=cuda_dev).to(dt)
        w = [torch.randint(-127, 128, (n, k), generator=g, device=cuda_dev, dtype=torch.int8) for _ in "gu"]
        s = [((torch.rand(n, generator=g, device=cuda_dev) + 0.5) * 1e-3).to(dt) for _ in "gu"]
        calls.append((x, w[0], s[0], w[1], s[1]) if glu else (x, w[0], s[0]))
    op = int8_gemm_swiglu if glu else int8_gemm
    want = [op(*a) for a in calls]
    for a, y in zip(calls, want):
        gate, *up = ((a[0].double() @ (q.double() * c.double()[:, None]).T).to(dt).double() for q, c in zip(a[1::2], a[2::2]))
        ref = gate / (1 + torch.exp(-gate)) * up[0] if glu else gate
        # fp32 accumulation may move a product across a rounding, no further: 2^-10 (fp16), 2^-7 (bf16) of the norm
        assert float((y.double() - ref).norm() / ref.norm()) <= (2.0**-10 if dt is torch.float16 else 2.0**-7)
    for _ in range(60):
        outs = []
        for _ in range(10):
            for a in calls:
                outs.append(op(*a))
                torch.cuda.synchronize(cuda_dev)
        assert all(torch.equal(y, want[i % 8]) for i, y in enumerate(outs))
