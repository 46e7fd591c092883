"""The same attention call gives the same bits every time, also started on an idle GPU, with other calls' tiles left in
shared memory."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,t,hq", [(128, 1, 16), (64, 8, 16), (128, 24, 16), (64, 16, 16)])  # 16, 32, 96 and 64 rows
def test_repeated_calls(cuda_dev, d, t, hq, dt):
    from blackwell_ops.decode import KVCacheInt8, tree_attention_int8

    h, page, b = 4, 16, 6
    lens = [4000, 3100, 2048, 900, 127, 1]
    cols = -(-(lens[0] + t) // page)
    g = torch.Generator(device=cuda_dev).manual_seed(d + t)
    calls = []
    for _ in range(4):
        k, v = (torch.randint(-127, 128, (b * cols, h, page, d), generator=g, device=cuda_dev, dtype=torch.int8) for _ in "kv")
        ks, vs = ((torch.rand((b * cols, h, page), generator=g, device=cuda_dev) + 0.5) / 64 for _ in "kv")
        table = torch.randperm(b * cols, generator=g, device=cuda_dev).to(torch.int32).view(b, cols)
        q = torch.randn((b, t, hq, d), generator=g, device=cuda_dev).to(dt)
        calls.append((q, KVCacheInt8(k, v, ks, vs), table, torch.tensor(lens, dtype=torch.int32, device=cuda_dev)))
    want = [tree_attention_int8(*a) for a in calls]
    for _ in range(30):
        outs = []
        for _ in range(10):
            for a in calls:
                outs.append(tree_attention_int8(*a))
                torch.cuda.synchronize(cuda_dev)
        assert all(torch.equal(y, want[i % 4]) for i, y in enumerate(outs))
