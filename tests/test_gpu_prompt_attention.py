"""GPU parity of causal attention over packed prompts against the CPU oracle (oracle/prompt.py).

Tolerances, with A the sum of |v| by weight and B the largest sum of |scale q k| over a product's terms.  A score is
accumulated in fp32, sixteen products a step, D / 16 <= 16 steps, each off by 2^-23 of B at most: 2^-19 B, and a weight
relative to the others twice that, 2^-18 B.  A weight's exponential (2^-21 of it with its argument's rounding) and its
rounding to the inputs' type (half an ulp, u), the sum over n keys in n / 16 steps of 2^-23 each: all relative to A.  The
result is rounded once more: u of it, and 2^-25, half of fp16's smallest step."""
import numpy as np
import pytest

from oracle import prompt as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def _randn(seed, shape, dt, dev, spread=1.0):
    return (spread * torch.randn(shape, generator=torch.Generator().manual_seed(seed))).to(dt).to(dev)


def _off(lens, dev, first=0):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]) + first, dtype=torch.int32, device=dev)


def _check(q, k, v, offsets, scale=None, got=None):
    from blackwell_ops.prompt import prompt_attention

    got = prompt_attention(q, k, v, offsets, scale) if got is None else got
    assert got.shape == q.shape and got.dtype == q.dtype and got.is_contiguous()
    off = offsets.cpu().numpy()
    host = [x.float().cpu().numpy() for x in (q, k, v)]
    want, size, prod = ref.attention(*host, off, q.shape[-1] ** -0.5 if scale is None else scale)
    y = got.float().cpu().numpy().astype(np.float64)
    fine = np.isfinite(want) & np.isfinite(size) & np.isfinite(prod)
    assert np.isfinite(y[fine]).all()
    n = int((off[1:] - off[:-1]).max(initial=0))
    u = U[q.dtype]
    bound = u * np.abs(want) + 2.0**-25 + size * (u + 2.0**-20 + (n / 16 + 8) * 2.0**-23 + 2.0**-18 * prod)
    err = np.abs(y - want)
    assert (err[fine] <= bound[fine]).all(), (float((err - bound)[fine].max()), np.argwhere(fine & (err > bound))[:4].tolist())
    none = np.ones(len(y), dtype=bool)
    none[off[0]:off[-1]] = False
    assert not y[none].any()
    return got


HEADS = [(1, 1, 128), (128, 1, 64), (100, 1, 128), (16, 8, 128), (32, 8, 128), (28, 4, 64), (12, 1, 128), (8, 8, 64), (64, 8, 64), (5, 1, 64)]
ODD = [(4, 2, 80), (3, 3, 96), (2, 1, 256), (2, 2, 1), (6, 2, 33), (130, 1, 32), (130, 1, 64), (4, 4, 192)]
LENS = [[1], [17], [0, 1, 2, 0, 3], [128], [127, 129], [16, 15, 14, 13, 33], [300, 0, 513], [64] * 9]


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hk,d", HEADS + ODD)
def test_shapes(cuda_dev, hq, hk, d, dt):
    for i, lens in enumerate(LENS if hq < 64 else LENS[:6]):
        n = sum(lens)
        q, k, v = (_randn(10 * i + s, (n, h, d), dt, cuda_dev, x) for s, h, x in ((1, hq, 2.5), (2, hk, 1), (3, hk, 1)))
        _check(q, k, v, _off(lens, cuda_dev))


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hk,d", [(16, 8, 128), (28, 4, 64), (12, 1, 128), (4, 2, 80)])
def test_rows_of_no_sequence(cuda_dev, hq, hk, d, dt):
    """Spare rows before the first and behind the last sequence, with anything in them, give zeros and touch no other."""
    for lens, first, last in (([5], 0, 3), ([130, 0, 7], 9, 300), ([1, 1], 1, 129), ([], 0, 40), ([0, 0], 3, 5)):
        n = sum(lens) + first + last
        q, k, v = (_randn(s, (n, h, d), dt, cuda_dev) for s, h in ((1, hq), (2, hk), (3, hk)))
        off = _off(lens, cuda_dev, first)
        want = _check(q, k, v, off)
        for x in (q, k, v):
            x[:first], x[n - last:] = float("nan"), float("inf")
        _check(q, k, v, off, got=want)
        from blackwell_ops.prompt import prompt_attention

        assert torch.equal(prompt_attention(q, k, v, off), want)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hk,d", [(16, 8, 128), (28, 4, 64), (4, 2, 80)])
def test_what_is_not_seen(cuda_dev, hq, hk, d, dt):
    """NaN and infinities in later rows, and in other sequences, change nothing before them."""
    from blackwell_ops.prompt import prompt_attention

    lens = [200, 77, 300]
    off, n = _off(lens, cuda_dev), sum(lens)
    q, k, v = (_randn(s, (n, h, d), dt, cuda_dev) for s, h in ((1, hq), (2, hk), (3, hk)))
    want = _check(q, k, v, off)
    for at in (1, 63, 127, 128, 130, 199):
        for x in (q, k, v):
            for bad in (float("nan"), float("inf"), -float("inf")):
                y = x.clone()
                y[at, 0, d // 2] = bad
                got = prompt_attention(*(y if z is x else z for z in (q, k, v)), off)
                assert torch.equal(got[:at], want[:at]) and torch.equal(got[200:], want[200:]), (at, bad)
                grp = hq // hk if x is not q else 1
                assert torch.equal(got[:, grp:], want[:, grp:])
                if x is v:  # seen by every later row, in this element alone
                    seen = got[at:200, :grp, d // 2]
                    assert bool((seen.isnan() if bad != bad else seen == bad).all()), (at, bad)
                    rest = torch.arange(d, device=cuda_dev) != d // 2
                    assert torch.equal(got[:, :grp][..., rest], want[:, :grp][..., rest])
    # infinities of both signs in one column: NaN from the second on
    y = v.clone()
    y[140, 0, 3], y[150, 0, 3] = float("inf"), -float("inf")
    got = prompt_attention(q, k, y, off)
    assert bool((got[140:150, 0, 3] == float("inf")).all()) and bool(got[150:200, 0, 3].isnan().all())
    assert torch.equal(got[:140], want[:140]) and torch.equal(got[200:], want[200:])


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128, 80])
def test_scores_that_grow(cuda_dev, d, dt):
    """Every tile has larger scores than the one before, so a row's reference moves; or far smaller ones."""
    n = 700
    q, k, v = (_randn(s, (n, h, d), dt, cuda_dev) for s, h in ((1, 4), (2, 2), (3, 2)))
    ramp = torch.linspace(0, 1, n, device=cuda_dev)[:, None, None]
    u = torch.nn.functional.normalize(_randn(7, (1, 1, d), torch.float32, cuda_dev), dim=-1)
    for sign, size in ((1, 60.0), (-1, 60.0), (1, 400.0)):
        kk = (k.float() * 0.2 + sign * ramp * size * u).to(dt)
        qq = (q.float() * 0.2 + d ** 0.5 * u).to(dt)
        _check(qq, kk, v, _off([n], cuda_dev))
        _check(qq, kk, v, _off([n - 260, 260], cuda_dev))


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hk,d", [(4, 2, 128), (4, 2, 64), (4, 2, 80)])
def test_the_largest_and_smallest_values(cuda_dev, hq, hk, d, dt):
    """Values up to half the type's largest, whose mean is in range where their sum is not; and tiny ones."""
    q, k = (_randn(s, (700, h, d), dt, cuda_dev) for s, h in ((1, hq), (2, hk)))
    v = torch.rand((700, hk, d), generator=torch.Generator().manual_seed(3)).to(cuda_dev) * 0.5 + 0.5
    _check(q, k, (v * (torch.finfo(dt).max / 2)).to(dt), _off([1, 2, 97, 600], cuda_dev))
    _check(q, k, (v * 2.0**-14).to(dt), _off([1, 2, 97, 600], cuda_dev))


def test_scales(cuda_dev):
    q, k, v = (_randn(s, (300, h, 128), torch.bfloat16, cuda_dev) for s, h in ((1, 8), (2, 2), (3, 2)))
    off = _off([300], cuda_dev)
    for scale in (0.0, -0.3, 1.0, 0.01):
        _check(q, k, v, off, scale)


@pytest.mark.parametrize("hq,hk,d", [(16, 8, 128), (28, 4, 64), (4, 2, 80)])
def test_strides(cuda_dev, hq, hk, d):
    lens = [150, 33]
    n = sum(lens)
    off = _off(lens, cuda_dev)
    qkv = _randn(1, (n, hq + 2 * hk, d), torch.float16, cuda_dev)
    q, k, v = qkv.split([hq, hk, hk], dim=1)
    want = _check(q, k, v, off)
    by_head = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]       # heads outermost
    wide = _randn(2, (n, hq + 2 * hk, d + 3), torch.float16, cuda_dev)                   # rows that start anywhere
    wide[..., 3:] = qkv
    odd = wide[..., 3:].split([hq, hk, hk], dim=1)
    every = qkv.new_zeros((n, hq + 2 * hk, 2 * d))                                       # every other element
    every[..., ::2] = qkv
    from blackwell_ops.prompt import prompt_attention

    for x in (by_head, odd, every[..., ::2].split([hq, hk, hk], dim=1)):
        assert torch.equal(prompt_attention(*x, off), want)
    one = k[:, :1].expand(n, hk, d)                                                      # one key head for all
    _check(q, one, v, off)
    row = v[:1].expand(n, hk, d)                                                         # one row of values
    _check(q, k, row, off)
    slack = torch.zeros(7, dtype=torch.int32, device=cuda_dev)
    slack[1::2] = off
    assert torch.equal(prompt_attention(q, k, v, slack[1::2]), want)


def test_alone_and_together(cuda_dev):
    """A sequence's results do not depend on the others, and are the same in every run."""
    from blackwell_ops.prompt import prompt_attention

    for hq, hk, d in ((16, 8, 128), (28, 4, 64)):
        lens = [1, 700, 0, 129, 40, 1500, 3]
        off, n = _off(lens, cuda_dev), sum(lens)
        q, k, v = (_randn(s, (n, h, d), torch.bfloat16, cuda_dev) for s, h in ((1, hq), (2, hk), (3, hk)))
        want = prompt_attention(q, k, v, off)
        at = 0
        for m in lens:
            s = slice(at, at + m)
            assert torch.equal(prompt_attention(q[s], k[s], v[s], _off([m], cuda_dev)), want[s])
            at += m
        for _ in range(20):
            assert torch.equal(prompt_attention(q, k, v, off), want)


def test_long(cuda_dev):
    """A long prompt against the definition in 64 bits on the device."""
    for dt, hq, hk, d, n in ((torch.bfloat16, 4, 2, 128, 9001), (torch.float16, 7, 1, 64, 6000)):
        from blackwell_ops.prompt import prompt_attention

        q, k, v = (_randn(s, (n, h, d), dt, cuda_dev, x) for s, h, x in ((1, hq, 2.5), (2, hk, 1), (3, hk, 1)))
        got = prompt_attention(q, k, v, _off([n], cuda_dev)).double()
        u = U[dt]
        for h in range(hq):
            kk, vv = k[:, h // (hq // hk)].double(), v[:, h // (hq // hk)].double()
            z = (q[:, h].double() @ kk.T * d ** -0.5).masked_fill(torch.ones((n, n), dtype=torch.bool, device=cuda_dev).triu(1), -float("inf"))
            p = z.softmax(-1)
            want, size = p @ vv, p @ vv.abs()
            prod = (q[:, h].double().abs() @ kk.abs().T * d ** -0.5).amax(-1, keepdim=True)
            bound = u * want.abs() + 2.0**-25 + size * (u + 2.0**-20 + (n / 16 + 8) * 2.0**-23 + 2.0**-18 * prod)
            assert bool(((got[:, h] - want).abs() <= bound).all())


def test_streams_and_graphs(cuda_dev):
    """Captured once, replayed with other lengths and inputs on another stream."""
    from blackwell_ops.prompt import prompt_attention

    n = 400
    q, k, v = (_randn(s, (n, h, 128), torch.bfloat16, cuda_dev) for s, h in ((1, 16), (2, 8), (3, 8)))
    off = _off([150, 30, 220], cuda_dev)
    g, h = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = prompt_attention(q, k, v, off)
    with torch.cuda.graph(h):
        twice = prompt_attention(out, k, v, off)
    off.copy_(_off([0, 391, 2], cuda_dev))
    q.copy_(_randn(9, (n, 16, 128), torch.bfloat16, cuda_dev))
    st = torch.cuda.Stream(cuda_dev)
    st.wait_stream(torch.cuda.current_stream(cuda_dev))
    with torch.cuda.stream(st):
        g.replay()
        h.replay()
        mine = prompt_attention(prompt_attention(q, k, v, off), k, v, off)
    st.synchronize()
    assert torch.equal(twice, mine)
    _check(q, k, v, off, got=out)


def test_offsets_out_of_order_stay_inside(cuda_dev):
    """Offsets that descend or pass the rows: undefined results, nothing outside is read or written."""
    from blackwell_ops.prompt import prompt_attention

    for hq, hk, d in ((4, 2, 128), (4, 2, 80)):
        n = 300
        guard = torch.zeros((n + 2000, hq, d), dtype=torch.float16, device=cuda_dev)
        q, k, v = (_randn(s, (n, h, d), torch.float16, cuda_dev) for s, h in ((1, hq), (2, hk), (3, hk)))
        for off in ([0, 200, 100, 300], [5, 500, 1000, 2000], [-7, 3, -100, 12], [9, 8, 7, 6], [300, 0, 300, 0]):
            out = prompt_attention(q, k, v, torch.tensor(off, dtype=torch.int32, device=cuda_dev))
            assert out.shape == (n, hq, d)
        torch.cuda.synchronize()
        assert not bool(guard.any())


def test_refusals(cuda_dev):
    from blackwell_ops.prompt import prompt_attention

    q, k = (torch.zeros((6, h, 64), dtype=torch.float16, device=cuda_dev) for h in (4, 2))
    off = _off([2, 4], cuda_dev)
    for match, fn in [
        ("q must be CUDA", lambda: prompt_attention(q.cpu(), k, k, off)),
        ("fp16 or bf16", lambda: prompt_attention(q.float(), k.float(), k.float(), off)),
        (r"\[N, heads, D\]", lambda: prompt_attention(q[None], k[None], k[None], off)),
        ("leading dimensions", lambda: prompt_attention(q, k[:5], k[:5], off)),
        ("one dtype", lambda: prompt_attention(q, k.bfloat16(), k, off)),
        ("one dtype", lambda: prompt_attention(q, k, k.bfloat16(), off)),
        ("q's head dimension", lambda: prompt_attention(q, k[..., :32], k[..., :32], off)),
        ("q's head dimension", lambda: prompt_attention(q, k, k[:, :1], off)),
        ("a multiple", lambda: prompt_attention(q[:, :3], k, k, off)),
        ("a multiple", lambda: prompt_attention(q, k[:, :0], k[:, :0], off)),
        ("must be 1 to 256", lambda: prompt_attention(*(x.repeat(1, 1, 5) for x in (q, k, k)), off)),
        ("offsets must be int32", lambda: prompt_attention(q, k, k, off.long())),
        ("offsets must be int32", lambda: prompt_attention(q, k, k, off.cpu())),
        (r"offsets must be \[B", lambda: prompt_attention(q, k, k, off[None])),
        (r"offsets must be \[B", lambda: prompt_attention(q, k, k, off[:0])),
    ]:
        with pytest.raises(RuntimeError, match=match):
            fn()
    assert prompt_attention(q[:0], k[:0], k[:0], off).shape == (0, 4, 64)
    assert not bool(prompt_attention(q + 1, k + 1, k + 1, off[:1]).any())  # no sequence at all
