"""GPU parity of verify_tree against the oracle's walk: every accepted node and token equal.

The comparisons are 32-bit ones that both sides round alike; only the normaliser after a rejected sibling depends on the
order of a sum (2e-7 relative), so a decision could differ only for a random number that close to its threshold."""
import numpy as np
import pytest

from oracle import decode as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def _softmax(z):
    e = np.exp(z - z.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


def _case(seed, b, t, v, tree, drafts, sharp=2.0, noise=0.7):
    rng = np.random.default_rng(seed)
    z = rng.standard_normal((b, t, v)) * sharp
    p, q = _softmax(z), _softmax(z + noise * rng.standard_normal((b, t, v)))
    if tree == "chain":
        par = np.tile(np.arange(t) - 1, (b, 1))
    elif tree == "star":
        par = np.zeros((b, t), dtype=np.int64)
    else:
        par = np.array([[-1] + [rng.integers(max(0, i - 4), i) for i in range(1, t)] for _ in range(b)])
    par[:, 0] = -1
    tok = np.zeros((b, t), dtype=np.int64)
    for i in range(b):
        for j in range(1, t):
            tok[i, j] = np.argmax(q[i, par[i, j]] / rng.exponential(size=v))
    u, e = rng.random((b, t)).astype(np.float32), rng.exponential(size=(b, v)).astype(np.float32)
    return p, tok, par.astype(np.int32), u, e, q if drafts else None


def _run(case, dev):
    from blackwell_ops.decode import verify_tree

    p, tok, par, u, e, q = (None if x is None else torch.from_numpy(np.ascontiguousarray(x)).to(dev) for x in case)
    return verify_tree(p, tok, par, u, e, q)


def _check(case, dev):
    got, want = _run(case, dev), ref.verify(*case)
    for name, g, w in zip(("n", "path", "out"), got, want):
        g = g.cpu().numpy()
        assert g.dtype == w.dtype and np.array_equal(g, w), f"{name}: {np.argwhere(g != w)[:4].tolist()}"
    return want


@pytest.mark.parametrize("drafts", [True, False])
@pytest.mark.parametrize("b,t,v,tree", [(1, 1, 1, "chain"), (1, 1, 1000, "chain"), (3, 2, 7, "chain"), (40, 5, 100, "chain"),
                                        (2, 5, 50257, "chain"), (40, 8, 33, "star"), (30, 24, 257, "tree"), (7, 64, 1000, "tree"),
                                        (2, 64, 32001, "star"), (1, 9, 151936, "tree"), (5, 16, 4096, "tree"), (200, 3, 31, "star")])
def test_walks(cuda_dev, b, t, v, tree, drafts):
    n, _, _ = _check(_case(b * 100 + t, b, t, v, tree, drafts), cuda_dev)
    if b >= 40 and t > 2:
        assert n.max() > 0 and n.min() < t - 1  # both kinds of end were met


def test_padding_ties_and_empty_residuals(cuda_dev):
    b, t, v = 8, 6, 300
    p, tok, par, u, e, q = _case(1, b, t, v, "tree", True)
    par[0, 3:] = -1                                    # padded nodes
    par[1, 2], par[1, 4] = 2, 5                        # nodes that hang from themselves or later ones
    tok[2, 1], tok[2, 2], tok[2, 3] = -1, v, 2**40     # tokens that are none
    p[3], e[3] = 1.0 / v, 1.0                          # equal scores everywhere: the lowest token
    q[4] = p[4]                                        # p == q: nothing is left after a rejection ...
    u[4] = 1.0 - 2.0**-24
    p[5] = 0
    p[5, :, 17] = 1.0                                  # a target that is certain
    e[6, 9] = 0.0                                      # an exponential of zero
    u[7] = np.nan                                      # no number: never taken
    for drafts in (q, None):
        _check((p, tok, par, u, e, drafts), cuda_dev)
    # ... forced: the residual is empty, and the token comes from p
    u[4] = 2.0
    par[4] = [-1, 0, 0, 0, 0, 0]
    _check((p, tok, par, u, e, q), cuda_dev)
    p[6] = 0                                           # no candidate at all
    p[0, 0, 5] = np.nan
    _check((p, tok, par, u, e, q), cuda_dev)


@pytest.mark.parametrize("v", [4096, 4099, 200])
@pytest.mark.parametrize("b", [3, 20])
def test_scores_near_and_out_of_range(cuda_dev, b, v):
    """The last token is the best rounded quotient, lowest token first, where quotients are equal or a few ulps apart,
    within one thread's part and across parts, and where weights or exponentials are tiny, huge, zero, infinite or (the weights) NaN."""
    rng = np.random.default_rng(v + b)
    f = np.float32
    for kind in range(9):
        p, tok, par, u, e, q = _case(kind, b, 1, v, "chain", True)
        if kind == 0:                                 # two to five quotients a few ulps apart near the top
            for i in range(b):
                at = rng.choice(v, 5, replace=False)
                p[i, 0, at], e[i, at] = f(0.9), f(1e-3) * (1 + f(2.0**-23) * rng.integers(0, 9, 5).astype(f))
        elif kind == 1:                               # neighbours, the same quotient from different pairs
            p[:, 0, 8], e[:, 8] = f(0.25), f(2.0**-20)
            p[:, 0, 9], e[:, 9] = f(0.5), f(2.0**-19)
            p[:, 0, v - 1], e[:, v - 1] = f(0.125), f(2.0**-21)
        elif kind == 2:
            p *= f(1e-30)                             # all scores below the trusted range
        elif kind == 3:
            p *= f(1e-42)                             # subnormal weights
        elif kind == 4:
            e[:, 5] = f(1e-44)                        # a subnormal exponential: the quotient overflows or is huge
        elif kind == 5:
            e[:, 7], p[:, 0, 7] = 0.0, f(1e-3)        # infinite
            e[:, 11], p[:, 0, 11] = 0.0, 0.0          # no candidate
        elif kind == 6:
            e[:, 3] = np.inf
            p[:, 0, 6] = np.nan
        elif kind == 7:
            p[:, 0] = 0.0
            p[:, 0, v // 2], e[:, v // 2] = f(1e-20), f(1e25)   # the only candidate
        else:
            p *= f(1e30)
            e *= f(1e-25)
        with np.errstate(all="ignore"):
            _check((p, tok, par, u, e, q), cuda_dev)


def test_strides(cuda_dev):
    from blackwell_ops.decode import verify_tree

    case = _case(3, 4, 5, 501, "tree", True)
    want = ref.verify(*case)
    p, tok, par, u, e, q = (torch.from_numpy(np.ascontiguousarray(x)).to(cuda_dev) for x in case)
    wide = torch.empty((4, 5, 1003), device=cuda_dev)
    wide[..., 1:502] = p  # unaligned rows
    got = verify_tree(wide[..., 1:502], tok.t().contiguous().t(), par, u, e, q.transpose(0, 1).contiguous().transpose(0, 1))
    for g, w in zip(got, want):
        assert np.array_equal(g.cpu().numpy(), w)
    odd = torch.empty(4 * 5 * 501 + 3, device=cuda_dev)[3:].view(4, 5, 501).copy_(p)  # a base of 4-byte alignment
    for g, w in zip(verify_tree(odd, tok, par, u, e, q), want):
        assert np.array_equal(g.cpu().numpy(), w)


@pytest.mark.parametrize("tree,drafts", [("chain", True), ("star", True), ("star", False)])
def test_distribution(cuda_dev, tree, drafts):
    """The first token is distributed as the target's root row, whatever the drafts: 200000 walks, each frequency
    within 5 standard deviations (12 frequencies: one in 150000 such tests would fail by chance)."""
    from blackwell_ops.decode import verify_tree

    g = torch.Generator(device=cuda_dev).manual_seed(5)
    n, t, v = 200_000, 4, 12
    p = torch.softmax(torch.randn((t, v), generator=g, device=cuda_dev), -1)
    q = torch.softmax(torch.randn((t, v), generator=g, device=cuda_dev), -1)
    par = torch.tensor([-1, 0, 1, 2] if tree == "chain" else [-1, 0, 0, 0], dtype=torch.int32, device=cuda_dev)
    exp = torch.empty((n, t, v), device=cuda_dev).exponential_(generator=g)
    tok = (q[par.clamp(min=0).long()] / exp).argmax(-1)
    if not drafts:
        tok = torch.tensor([0, 3, 7, 1], device=cuda_dev).expand(n, t).contiguous()
    u = torch.rand((n, t), generator=g, device=cuda_dev)
    e = torch.empty((n, v), device=cuda_dev).exponential_(generator=g)
    _, _, out = verify_tree(p.expand(n, t, v), tok, par.expand(n, t).contiguous(), u, e,
                            q.expand(n, t, v) if drafts else None)
    freq = torch.bincount(out[:, 0], minlength=v).double() / n
    sd = (p[0].double() * (1 - p[0].double()) / n).sqrt()
    assert bool(((freq - p[0].double()).abs() <= 5 * sd).all()), ((freq - p[0].double()).abs() / sd).tolist()


def test_refusals(cuda_dev):
    from blackwell_ops.decode import verify_tree

    p = torch.ones((2, 3, 8), device=cuda_dev) / 8
    tok, par = torch.zeros((2, 3), dtype=torch.int64, device=cuda_dev), torch.zeros((2, 3), dtype=torch.int32, device=cuda_dev)
    u, e = torch.rand((2, 3), device=cuda_dev), torch.ones((2, 8), device=cuda_dev)
    for match, args in [
        ("CUDA fp32", (p.cpu(), tok, par, u, e)), ("CUDA fp32", (p.half(), tok, par, u, e)),
        (r"\[B, T, V\]", (p[0], tok, par, u, e)), (r"\[B, T, V\]", (p[..., :0], tok, par, u, e)),
        ("at most 64", (p[:, :1].expand(2, 65, 8), tok, par, u, e)), ("tokens must be", (p, tok.int(), par, u, e)),
        ("tokens must be", (p, tok[:1], par, u, e)), ("parents must be", (p, tok, par.long(), u, e)),
        ("accept_u must be", (p, tok, par, u[:, :2], e)), ("sample_e must be", (p, tok, par, u, e[:, :7])),
        ("draft_probs must be", (p, tok, par, u, e, p[:1])), ("draft_probs must be", (p, tok, par, u, e, p.half())),
    ]:
        with pytest.raises(RuntimeError, match=match):
            verify_tree(*args)
    n, path, out = verify_tree(p[:0], tok[:0], par[:0], u[:0], e[:0])
    assert n.shape == (0,) and path.shape == (0, 3) and out.shape == (0, 3)
    n, path, out = verify_tree(p[:, :0], tok[:, :0], par[:, :0], u[:, :0], e)
    assert n.tolist() == [0, 0] and out.shape == (2, 0)
