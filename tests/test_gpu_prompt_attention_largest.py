"""Values of the type's largest: a weighted mean never passes them, whatever the rounding of the weights to 16 bits makes of
it.  Every row is a mean of values of one size, so it is that value within the tolerance of test_gpu_prompt_attention (half
an ulp of the weights and of the result, and fp32 sums: under 2^-7 in bf16 and 2^-10 in fp16), and finite."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_prompt_attention import _off, _randn  # noqa: E402


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hk,d", [(4, 2, 128), (4, 2, 64), (4, 2, 80)])
def test_values_of_the_largest(cuda_dev, hq, hk, d, dt):
    from blackwell_ops.prompt import prompt_attention

    n, top = 700, torch.finfo(dt).max
    sign = torch.where(torch.arange(d, device=cuda_dev) % 2 == 0, 1.0, -1.0)
    v = (sign * top).to(dt).expand(n, hk, d).contiguous()
    u = torch.nn.functional.normalize(_randn(7, (1, 1, d), torch.float32, cuda_dev), dim=-1)
    for spread in (0.1, 1.0, 5.0):  # single keys that outweigh the rest by less than the reference's slack, and by more
        for seed in range(4):
            q = (_randn(seed, (n, hq, d), dt, cuda_dev).float() * 0.3 + d ** 0.5 * u).to(dt)
            k = (_randn(seed + 9, (n, hk, 1), torch.float32, cuda_dev) * spread * u).to(dt)
            for lens in ([n], [1, 2, 97, 600]):
                got = prompt_attention(q, k, v, _off(lens, cuda_dev))
                assert bool(got.isfinite().all()), int((~got.isfinite()).sum())
                slack = 2.0**-7 if dt is torch.bfloat16 else 2.0**-10
                assert bool(((got.double() / (sign.double() * top) - 1).abs() <= slack).all())
