"""The kernels' own search of blocks in the offsets: every row of many sequences is written once, by its sequence's block.

Keys of zeros weigh alike, so row p of a sequence of values 1, 2, .. is their mean (p + 2) / 2.  All weights are one number,
2^7 or 2^-16 within 2^-22 (the exponential's error); were it a power of two, the sums, whole numbers under 2^24 times it,
would be exact, so they are off by 2^-21 at most.  The reciprocal and the product add 2^-23, the result's rounding to fp16
2^-11."""
import random

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("hq,hk,d", [(2, 1, 64), (7, 1, 128), (16, 8, 128), (128, 1, 64), (2, 1, 20)])
@pytest.mark.parametrize("b", [0, 1, 2, 29, 30, 31, 32, 33, 63, 200, 1023, 1500])
def test_every_row_once(cuda_dev, b, hq, hk, d):
    from blackwell_ops.prompt import prompt_attention

    rng = random.Random(b)
    for trial in range(4 if b < 1000 else 2):
        p = rng.choice([16, 18, 64, 128, 256])
        most = 3 * p if b < 100 else 20
        lens = [rng.choice([0, 0, 1, 2, rng.randint(0, most), p if b < 100 else 3, p + 1 if b < 100 else 1]) for _ in range(b)]
        first, spare = rng.choice([0, 0, 3, p, 2 * p + 1]), rng.choice([0, 0, 5, p, 3 * p - 1])
        n = first + sum(lens) + spare
        place = torch.cat([torch.full((first,), -2.0), *(torch.arange(m, dtype=torch.float32) for m in lens),
                           torch.full((spare,), -2.0)]).to(cuda_dev)
        if n == 0:
            continue
        offsets = torch.tensor([first, *lens]).cumsum(0).to(torch.int32).to(cuda_dev)
        k = torch.zeros((n, hk, d), dtype=torch.float16, device=cuda_dev)
        v = torch.where(place < 0, 7.0, place + 1)[:, None, None].expand(n, hk, d).to(torch.float16).contiguous()
        got = prompt_attention(torch.ones((n, hq, d), dtype=torch.float16, device=cuda_dev), k, v, offsets).float()
        want = ((place + 2) / 2)[:, None, None]  # (0 for rows of no sequence)
        assert bool(((got - want).abs() <= want * (2.0**-11 + 2.0**-20)).all()), (trial, p, first, spare)
