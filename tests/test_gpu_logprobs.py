"""GPU parity of the log probabilities of given tokens against the CPU oracle (oracle/prompt.py).

Tolerances.  S is a sum of positive weights: a weight is off by 2^-22 (its exponential) and by |z| 2^-24 where its
exponent z is under 24 in what counts (1.5e-6), a thread adds at most 40 groups of eight (43 additions), the threads 20
more, each rounded by 2^-24 (4e-6): ln S is off by 6e-6, and so is a log probability, next to the rounding of x - m and of
the result (2^-23 of it).  T is a sum of terms of one sign with the same errors: the entropy ln S - T / S is off by 6e-6
twice, the second time T / S, which is at most the entropy.  Tokens are exact."""
import numpy as np
import pytest

from oracle import prompt as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def _check(x, tokens, top):
    from blackwell_ops.prompt import token_logprobs

    got = token_logprobs(x, tokens, top)
    want = ref.logprobs(x.float().cpu().numpy(), tokens.cpu().numpy(), min(top, x.shape[-1]))
    for y, w, slack in zip(got[:3], want[:3], (0, 1, 0)):
        y = y.cpu().numpy().astype(np.float64)
        assert y.shape == w.shape
        assert np.array_equal(np.isnan(y), np.isnan(w))
        finite = np.isfinite(w)
        assert np.array_equal(y[~finite & ~np.isnan(w)], w[~finite & ~np.isnan(w)])
        err = np.abs(y - w)[finite] if finite.any() else np.zeros(1)
        bound = 6e-6 * (1 + slack) + (2.0**-23 + 6e-6 * slack) * np.abs(w[finite]) if finite.any() else np.zeros(1)
        assert (err <= bound).all(), float((err - bound).max())
    assert got[3].dtype == torch.int64 and np.array_equal(got[3].cpu().numpy(), want[3])
    assert bool((got.entropy[~got.entropy.isnan()] >= 0).all())
    return got


def _logits(seed, rows, v, dt, dev, spread=4.0):
    return (spread * torch.randn((rows, v), generator=torch.Generator().manual_seed(seed))).to(dt).to(dev)


def _tokens(seed, rows, v, dev):
    t = torch.randint(0, v, (rows,), generator=torch.Generator().manual_seed(seed))
    if rows > 2:
        t[1], t[2] = -100, v
    return t.to(dev)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,v,top", [(1, 1, 1), (3, 2, 2), (5, 7, 20), (4, 8, 8), (4, 9, 3), (3, 33, 32), (9, 100, 0), (7, 511, 5),
                                        (3, 4095, 20), (2, 4096, 32), (2, 4097, 1), (5, 4104, 7), (300, 1000, 4), (33, 32000, 5),
                                        (3, 50257, 20), (1, 151936, 20), (17, 128256, 32), (160, 20001, 2)])
def test_shapes(cuda_dev, rows, v, top, dt):
    _check(_logits(rows + v, rows, v, dt, cuda_dev), _tokens(v, rows, v, cuda_dev), top)


@pytest.mark.parametrize("dt", DTYPES)
def test_ties(cuda_dev, dt):
    g = torch.Generator().manual_seed(1)
    for v in (10, 700, 5000, 37000):
        few = torch.randint(0, 4, (6, v), generator=g).to(dt)                     # four values
        few[1] = 0                                                               # one value
        few[2] = (torch.arange(v) % 4096).to(dt)                                 # every thread's groups alike
        few[3] = torch.arange(v).to(torch.float32).div(64).floor().to(dt)        # ascending
        few[4] = -few[3]
        few[5] = torch.where(torch.arange(v) % 2 == 0, -0.0, 0.0).to(dt)         # -0 is 0
        for top in (1, 5, 32):
            _check(few.to(cuda_dev), _tokens(v, 6, v, cuda_dev), top)


@pytest.mark.parametrize("dt", DTYPES)
def test_masked(cuda_dev, dt):
    """-inf and the type's lowest value, rows of nothing else, a single token, NaN and +inf in some rows."""
    for v in (5, 100, 3001, 40000):
        x = _logits(v, 16, v, dt, cuda_dev)
        low = torch.finfo(dt).min
        drop = torch.rand((16, v), generator=torch.Generator().manual_seed(2)).to(cuda_dev) < 0.97
        x[0], x[1] = -float("inf"), low
        x[2, :], x[2, v // 2] = -float("inf"), -7.5
        x[3, :], x[3, v - 1] = low, 3.0
        x[4] = x[4].masked_fill(drop[4], -float("inf"))
        x[5] = x[5].masked_fill(drop[5], low)
        x[6] = torch.where(drop[6], -float("inf"), low)
        x[7, v // 3] = float("nan")
        x[8, 0] = float("inf")
        x[9, v - 1], x[9, 0] = float("inf"), -float("inf")
        x[10] = float("nan")
        x[11] = torch.finfo(dt).max
        x[12, 1] = torch.finfo(dt).max
        x[13] = -float("inf")
        x[13, v - 1] = float("nan")
        for top in (0, 3, 32):
            tokens = _tokens(3, 16, v, cuda_dev)
            tokens[5:] = torch.arange(11, device=cuda_dev) % v
            _check(x, tokens, top)


@pytest.mark.parametrize("dt", DTYPES)
def test_large_differences(cuda_dev, dt):
    """Peaked rows, and logits far from zero (their differences count)."""
    x = _logits(5, 8, 9001, dt, cuda_dev, 60.0)
    x[3:] = (x[3:].float() / 200 + 3000).to(dt)
    _check(x, _tokens(6, 8, 9001, cuda_dev), 10)


@pytest.mark.parametrize("dt", DTYPES)
def test_strides_and_leading_dimensions(cuda_dev, dt):
    from blackwell_ops.prompt import token_logprobs

    x = _logits(8, 12, 3000, dt, cuda_dev)
    t = _tokens(9, 12, 2000, cuda_dev)
    for off in range(9):  # rows that start anywhere
        _check(x[:, off:2000 + off], t, 6)
        _check(x[::2, off:2000 + 2 * off], t[::2], 3)
    _check(x[:, ::3], t.clamp(max=999), 5)
    _check(x.T[:12, :12], t, 4)
    _check(x[:1].expand(12, 3000), t, 4)  # one row, twelve times
    want = token_logprobs(x, t, 7)
    for got, w in zip(token_logprobs(x.view(3, 4, 3000), t.view(3, 4), 7), want):
        assert torch.equal(got.flatten(0, 1), w)
    for got, w in zip(token_logprobs(x[4], t[4], 7), want):
        assert torch.equal(got, w[4])
    assert token_logprobs(x[:0], t[:0], 5).top_tokens.shape == (0, 5)
    assert token_logprobs(x.view(3, 4, 3000)[:, :0], t.view(3, 4)[:, :0], 5).top_logprobs.shape == (3, 0, 5)


def test_rows_alone_and_together(cuda_dev):
    """A row's results do not depend on how many rows there are."""
    from blackwell_ops.prompt import token_logprobs

    for dt in DTYPES:
        for v in (3000, 151936):
            x, t = _logits(3, 300, v, dt, cuda_dev), torch.arange(300, device=cuda_dev)
            for top in (0, 20):
                want = token_logprobs(x, t, top)
                for n in (1, 2, 9, 18, 19, 37, 74, 75, 148, 149):
                    assert all(torch.equal(a, b[:n]) for a, b in zip(token_logprobs(x[:n], t[:n], top), want)), (n, top)
                assert all(torch.equal(a, b) for a, b in zip(token_logprobs(x, t, top), want))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,v", [(2, 16383), (2, 16384), (20, 16391), (28, 16400), (30, 16385), (50, 32767), (100, 32768), (120, 33001),
                                    (222, 32773), (223, 32770), (92, 62501), (93, 62500)])
def test_rows_of_one_two_and_four_ctas(cuda_dev, rows, v, dt):
    """At the lengths and numbers of rows where a row's CTAs change: ties across them, masked parts, a NaN in the last group."""
    x = _logits(rows + v, rows, v, dt, cuda_dev)
    x[0] = (torch.arange(v, device=cuda_dev) % 5).to(dt)
    x[1] = -float("inf")
    x[1, v - 3:] = 1.0
    x[rows // 2, :v - v // 4] = torch.finfo(dt).min
    if rows > 2:
        x[rows - 1, v - 1] = float("nan")
    _check(x, _tokens(v, rows, v, cuda_dev), 1)
    _check(x, _tokens(v, rows, v, cuda_dev), 20)


def test_many_rows(cuda_dev):
    """More rows than a grid's second dimension; offsets past 2^31 elements."""
    from blackwell_ops.prompt import token_logprobs

    x = _logits(1, 70000, 40, torch.float16, cuda_dev)
    _check(x, torch.arange(70000, device=cuda_dev) % 40, 2)
    big = torch.zeros((9000, 256000), dtype=torch.float16, device=cuda_dev)
    assert big.numel() > 2**31
    big[8999, 255999], big[8998, 7] = 9.0, 9.0
    got = token_logprobs(big, torch.full((9000,), 255999, device=cuda_dev), 2)
    assert got.top_tokens[8997:].tolist() == [[0, 1], [7, 0], [255999, 0]]
    lse = np.log(np.exp(9.0) + 255999)
    assert abs(float(got.logprobs[8999]) - (9 - lse)) <= 1e-5 and abs(float(got.logprobs[8998]) + lse) <= 1e-5


def test_streams_and_graphs(cuda_dev):
    from blackwell_ops.prompt import token_logprobs

    x, t = _logits(1, 5, 50257, torch.bfloat16, cuda_dev), torch.arange(5, device=cuda_dev)
    token_logprobs(x, t, 20)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = token_logprobs(x, t, 20)
    x.copy_(_logits(2, 5, 50257, torch.bfloat16, cuda_dev))
    st = torch.cuda.Stream(cuda_dev)
    st.wait_stream(torch.cuda.current_stream(cuda_dev))
    with torch.cuda.stream(st):
        g.replay()
        mine = token_logprobs(x, t, 20)
    st.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, mine))
    _check(x, t, 20)


def test_refusals(cuda_dev):
    from blackwell_ops.prompt import token_logprobs

    x, t = torch.zeros((3, 50), dtype=torch.float16, device=cuda_dev), torch.zeros(3, dtype=torch.int64, device=cuda_dev)
    for match, fn in [
        ("must be CUDA", lambda: token_logprobs(x.cpu(), t.cpu())),
        ("fp16, bf16 or fp32", lambda: token_logprobs(x.double(), t)),
        ("fp16, bf16 or fp32", lambda: token_logprobs(x.long(), t)),
        (r"\[\.\., V\]", lambda: token_logprobs(x[:, :0], t)),
        ("tokens must be int64", lambda: token_logprobs(x, t.int())),
        ("tokens must be int64", lambda: token_logprobs(x, t[:2])),
        ("tokens must be int64", lambda: token_logprobs(x, t.cpu())),
        ("top must be", lambda: token_logprobs(x, t, 33)),
        ("top must be", lambda: token_logprobs(x, t, -1)),
    ]:
        with pytest.raises(RuntimeError, match=match):
            fn()
