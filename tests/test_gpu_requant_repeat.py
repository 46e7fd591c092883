"""Merges and requantisations repeated from an idle GPU, several adapters in turn: the same bits every time."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("r", [8, 16, 40, 64, 128])
def test_repeated_calls(cuda_dev, r):
    from blackwell_ops.cuda import lora_merge, lora_merge_requant

    n, k = 2048, 2048
    g = torch.Generator(device=cuda_dev).manual_seed(r)
    args = [(torch.randn((n, k), generator=g, device=cuda_dev).half(), torch.randn((r, k), generator=g, device=cuda_dev).half(),
             torch.randn((n, r), generator=g, device=cuda_dev).half() * 0.02, 0.5) for _ in range(4)]
    want = [(*lora_merge_requant(*a), lora_merge(*a)) for a in args]
    for _ in range(25):
        outs = []
        for _ in range(10):
            for i, a in enumerate(args):
                outs.append((i, lora_merge_requant(*a), lora_merge(*a)))
                torch.cuda.synchronize(cuda_dev)
        for i, (q, s), m in outs:
            assert torch.equal(q, want[i][0]) and torch.equal(s, want[i][1]) and torch.equal(m, want[i][2])
