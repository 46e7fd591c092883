"""Values that are not finite: an element of v that is infinite or NaN goes to that element of every row that sees it,
whatever its weight (also one that underflows, and where all scores are -inf); nothing else changes by a bit, and nothing
of it depends on the other sequences, whose number decides how long the kernel's blocks are."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_prompt_attention import _check, _off, _randn  # noqa: E402

INF, NAN = float("inf"), float("nan")


def _same(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a[~a.isnan()], b[~b.isnan()])


def _passed(v, lens, hq):
    """Sums of the values that are not finite and that a row sees, 0 where there are none: [N, Hq, D]."""
    bad = torch.where(v.isfinite(), torch.zeros_like(v), v).float()
    at, out = 0, []
    for n in lens:
        out.append(bad[at:at + n].cumsum(0))
        at += n
    return torch.cat(out).repeat_interleave(hq // v.shape[1], dim=1)


def _inputs(kind, n, hq, hk, d, dt, dev):
    q, k, v = (_randn(s, (n, h, d), dt, dev) for s, h in ((1, hq), (2, hk), (3, hk)))
    u = torch.nn.functional.normalize(_randn(7, (1, 1, d), torch.float32, dev), dim=-1)
    ramp = (torch.arange(n, device=dev) % 701 / 700)[:, None, None]
    if kind in ("rising", "falling"):  # later keys far above earlier ones, whose weights underflow; or far below
        sign = 1 if kind == "rising" else -1
        k = (k.float() * 0.2 + sign * ramp * 400 * u).to(dt)
        q = (q.float() * 0.2 + d ** 0.5 * u).to(dt)
    return q, k, v


def _spoil(v, lens):
    at = 0
    for i, n in enumerate(lens):
        for j, (key, col, bad) in enumerate([(0, 0, INF), (5, 1, -INF), (130, 0, -INF), (130, 2, NAN), (300, 3, INF), (520, 3, INF),
                                             (520, -1, -INF), (n - 1, 5, INF)]):
            if key < n and (i + j) % 3 != 2:
                v[at + key, (i + j) % v.shape[1], col] = bad
        at += n
    return v


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind", ["plain", "rising", "falling"])
@pytest.mark.parametrize("hq,hk,d", [(4, 2, 128), (28, 4, 64), (3, 3, 128), (4, 2, 80)])
def test_values_that_are_not_finite(cuda_dev, hq, hk, d, kind, dt):
    from blackwell_ops.prompt import prompt_attention

    for lens in ([701], [701, 0, 129, 1, 640], [257] * 5, [701, 128, 256] * 30 if d != 80 else [130] * 40):
        n, off = sum(lens), _off(lens, cuda_dev)
        q, k, clean = _inputs(kind, n, hq, hk, d, dt, cuda_dev)
        v = _spoil(clean.clone(), lens)
        zeros = torch.where(v.isfinite(), v, torch.zeros_like(v))
        want = prompt_attention(q, k, zeros, off)
        if n < 3000 and kind == "plain":
            _check(q, k, zeros, off, got=want)
        passed = _passed(v, lens, hq)
        want = torch.where(passed == 0, want, passed.to(dt))
        got = prompt_attention(q, k, v, off)
        assert _same(got, want), (lens[:3], (got.isnan() != want.isnan()).sum())
        at = 0
        for m in lens[:8]:
            s = slice(at, at + m)
            assert _same(prompt_attention(q[s], k[s], v[s], _off([m], cuda_dev)), got[s])
            at += m


@pytest.mark.parametrize("hq,hk,d", [(4, 2, 128), (4, 2, 64), (4, 2, 80)])
def test_no_weight_at_all(cuda_dev, hq, hk, d):
    """Scores of -inf alone: zeros, but for what is not finite; scores with a NaN: NaN."""
    from blackwell_ops.prompt import prompt_attention

    n, off = 400, _off([400], cuda_dev)
    q = torch.full((n, hq, d), 1e30, dtype=torch.bfloat16, device=cuda_dev)
    k = torch.full((n, hk, d), -1e30, dtype=torch.bfloat16, device=cuda_dev)
    v = _randn(3, (n, hk, d), torch.bfloat16, cuda_dev)
    assert not bool(prompt_attention(q, k, v, off).any())
    v[3, 0, 7], v[200, 1, 8], v[250, 1, 8] = INF, -INF, NAN
    assert _same(prompt_attention(q, k, v, off).float(), _passed(v, [n], hq))
    q, k, _ = _inputs("plain", n, hq, hk, d, torch.bfloat16, cuda_dev)
    q[150, 0, 0] = NAN
    got = prompt_attention(q, k, v, off)
    assert bool(got[150, 0].isnan().all()) and bool((got[149:152, 0, 7][[0, 2]] == INF).all())
    rest = torch.ones(n, dtype=torch.bool, device=cuda_dev)
    rest[150] = False
    q[150, 0, 0] = 0
    assert _same(got[rest], prompt_attention(q, k, v, off)[rest])


def test_many_values_that_are_not_finite(cuda_dev):
    """All of v, in a long prompt: every row NaN or infinite, in a time near that of a clean one."""
    from blackwell_ops import _lib
    from blackwell_ops.prompt import prompt_attention

    n, off = 5000, _off([5000], cuda_dev)
    for d, dt in ((128, torch.bfloat16), (64, torch.float16)):
        q, k, v = (_randn(s, (n, 4, d), dt, cuda_dev) for s in (1, 2, 3))
        for bad in (INF, -INF, NAN):
            got = prompt_attention(q, k, torch.full_like(v, bad), off)
            assert bool((got.isnan() if bad != bad else got == bad).all())
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
