"""A row's log probabilities, bit for bit, wherever the row lies: behind any number of others, at any address, in a
cluster of one, two or four CTAs.  (Sums go by the logits' numbers; tolerances are those of test_gpu_logprobs.)"""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_logprobs import DTYPES, _check, _logits  # noqa: E402


def _alone(row, token, top):
    """The row in memory of its own, which starts on a boundary."""
    from blackwell_ops.prompt import token_logprobs

    one = row.clone()[None]
    assert one.data_ptr() % 256 == 0
    return token_logprobs(one, token[None], top)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("v", [1, 3, 7, 8, 9, 15, 16, 17, 23, 24, 25, 250, 257, 2047, 8191, 8193, 8197, 16385, 32771, 50257])
def test_equal_rows_anywhere(cuda_dev, v, dt):
    """One row many times: whatever precedes it (an odd vocabulary starts each row elsewhere), all results are the same."""
    from blackwell_ops.prompt import token_logprobs

    row = _logits(v, 1, v, dt, cuda_dev)[0]
    token = torch.tensor(v // 2, device=cuda_dev)
    for top in (0, 1, 20):
        want = _alone(row, token, top)
        for rows in (9, 33, 300):
            x = row.expand(rows, v).contiguous()
            for got, w in zip(token_logprobs(x, token.expand(rows), top), want):
                assert torch.equal(got, w.expand_as(got)), (rows, top)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("v", [5, 1003, 20001, 40007])
def test_rows_at_any_address(cuda_dev, v, dt):
    """Rows of a wider matrix whose other columns are NaN, from every start; masked rows and ties among them."""
    from blackwell_ops.prompt import token_logprobs

    x = _logits(v, 7, v, dt, cuda_dev)
    x[1] = -float("inf")
    x[2] = (torch.arange(v, device=cuda_dev) % 3).to(dt)
    x[3, : v - 1] = -float("inf")
    x[4, ::2] = torch.finfo(dt).min
    x[5, v // 2] = float("nan")
    token = torch.arange(7, device=cuda_dev) * (v // 7)
    want = [_alone(r, t, 6) for r, t in zip(x, token)]
    want = [torch.cat(y) for y in zip(*want)]
    for at in range(17):
        for pad in (17, 18, 24):
            wide = torch.full((7, v + pad), float("nan"), dtype=dt, device=cuda_dev)
            part = wide[:, at:at + v]
            part.copy_(x)
            for got, w in zip(token_logprobs(part, token, 6), want):
                assert torch.equal(got.nan_to_num(nan=7.0, posinf=1e9, neginf=-1e9), w.nan_to_num(nan=7.0, posinf=1e9, neginf=-1e9)), (at, pad)
            if pad == 17:
                _check(part, token, 6)


@pytest.mark.parametrize("dt", DTYPES)
def test_every_length_and_start(cuda_dev, dt):
    """Short rows of every length from every start, in memory whose other elements are +inf: each against the definition."""
    for v in range(1, 50):
        flat = torch.full((9 * (v + 9) + 64,), float("inf"), dtype=dt, device=cuda_dev)
        x = flat.as_strided((9, v), (v + 9 if v % 8 else v + 1, 1), 5)
        x.copy_(_logits(v, 9, v, dt, cuda_dev))
        _check(x, torch.arange(9, device=cuda_dev) % v, 4)
