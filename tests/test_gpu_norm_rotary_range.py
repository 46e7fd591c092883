"""The range of the norms of heads: squares are summed in fp32, so bf16 rows are right as long as that sum is in range, and
rows beyond it give zeros, as the interface says; their neighbours are as they were.

Tolerances as in test_gpu_norm_rotary: every square of a listed size is a normal number, so the same roundings count."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_norm_rotary import _near  # noqa: E402
from test_gpu_rotary_kv import _randn  # noqa: E402

# (without eps the sum has to be a normal number itself; 256 values of 5e17, 3.9 times that at most: under 2e38)
SIZES = [(1e-16, 0.0), (1e-8, 0.0), (1.0, 0.0), (5e17, 0.0), (1e-30, 1e-6), (1e-3, 1e-6), (1e12, 1e-6), (5e17, 1e-6)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot,first", [(128, 128, 0), (128, 64, 0), (64, 64, 0), (256, 256, 0), (32, 32, 0), (128, 128, 1), (80, 40, 0),
                                         (33, 2, 0)])
def test_large_and_tiny_rows(cuda_dev, d, rot, first, interleaved):
    """Every size beside every other, in rows of both kernels (``first``: rows that start on no 16-byte boundary)."""
    from blackwell_ops.decode import norm_rotary, rotary_frequencies, rotary_plan

    plan, (freq, mag) = rotary_plan(rot, interleaved=interleaved, device=cuda_dev), rotary_frequencies(rot)
    w = 1 + _randn(2, (d,), torch.bfloat16, cuda_dev) / 4
    pos = torch.arange(3, dtype=torch.int32, device=cuda_dev) * 1000
    for eps in sorted({e for _, e in SIZES}):
        sizes = [x for x, e in SIZES if e == eps]
        wide = torch.zeros((3, len(sizes), d + 8), dtype=torch.bfloat16, device=cuda_dev)
        x = wide[..., first:first + d]
        x.copy_(_randn(3, (3, len(sizes), d), torch.bfloat16, cuda_dev).clamp(-3.9, 3.9).float()
                * torch.tensor(sizes, device=cuda_dev)[:, None])
        for y in norm_rotary(x, x, pos, plan, w, w, eps=eps):
            _near(y, x, w, eps, pos.cpu().numpy(), plan, freq.numpy(), mag, interleaved, torch.bfloat16)


@pytest.mark.parametrize("d,rot", [(128, 128), (80, 40)])
def test_rows_beyond_the_range(cuda_dev, d, rot):
    """Zeros, in the cache too; the other heads and tokens as without them."""
    from blackwell_ops.decode import KVCacheInt8, norm_rotary_kv_write_int8, rotary_plan

    n, h = 9, 4
    plan, pos = rotary_plan(rot, device=cuda_dev), torch.arange(n, dtype=torch.int32, device=cuda_dev)
    w = 1 + _randn(5, (d,), torch.bfloat16, cuda_dev) / 4
    table, start = torch.zeros((1, 1), dtype=torch.int32, device=cuda_dev), torch.zeros(1, dtype=torch.int32, device=cuda_dev)
    off = torch.tensor([0, n], dtype=torch.int32, device=cuda_dev)
    x = _randn(1, (n, h, d), torch.bfloat16, cuda_dev)
    large = x.clone()
    large[::2, 1], large[3, 2, 5] = 1e25, torch.finfo(torch.bfloat16).max
    out = []
    for y in (x, large):
        cache = KVCacheInt8.empty(1, h, 16, d, device=cuda_dev)
        q, k = norm_rotary_kv_write_int8(y, y, x, pos, plan, cache, table, start, w, w, offsets=off, keys=True)
        out.append((q, k, cache.k[0].movedim(0, 1)[:n], cache.k_scale[0].movedim(0, 1)[:n, :, None], cache.v, cache.v_scale))
    beyond = (large != x).any(-1)
    assert int(beyond.sum()) == 6
    for a, b in list(zip(*out))[:4]:
        assert not bool(b[beyond].any()) and torch.equal(a[~beyond], b[~beyond])
    for a, b in list(zip(*out))[4:]:
        assert torch.equal(a, b)
