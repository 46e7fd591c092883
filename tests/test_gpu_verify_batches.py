"""verify_tree decides for a sequence as it does alone, whatever its batch: also where the normaliser's last bit decides."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("drafts", [True, False])
@pytest.mark.parametrize("v", [4096, 32001, 151936])
def test_same_alone_and_in_a_batch(cuda_dev, v, drafts):
    """The root's first child is rejected, the second one's random number is swept in steps of an ulp over the place where
    it is just accepted: u * draft * Z = w, Z summed over the row."""
    from blackwell_ops.decode import verify_tree

    f, steps = np.float32, np.arange(-20, 21)
    for seed in range(6):
        rng = np.random.default_rng(1000 * seed + v)
        p, q = (rng.exponential(size=v) ** 2 for _ in "pq")
        p, q = (p / p.sum()).astype(f), (q / q.sum()).astype(f)
        if drafts:
            w = np.maximum(p - q, f(0))
            first, second = int(np.argmin(p - q)), int(np.argmax(p - q))
            edge = f(w[second]) / (q[second] * f(w.sum(dtype=np.float64)))
        else:
            second, first = np.argsort(p)[-2:]
            w = p.copy()
            w[first] = 0
            edge = f(w[second]) / f(w.sum(dtype=np.float64))
        b = len(steps)
        u = np.full((b, 3), 2.0, dtype=f)                        # 2: never accepted
        u[:, 2] = edge * (1 + steps * 2.0**-23)
        tok = torch.tensor([0, int(first), int(second)], device=cuda_dev).expand(b, 3).contiguous()
        par = torch.tensor([-1, 0, 0], dtype=torch.int32, device=cuda_dev).expand(b, 3).contiguous()
        rows = lambda x: torch.from_numpy(np.tile(x, (3, 1))).to(cuda_dev)[None].expand(b, 3, v)  # noqa: E731
        pt, qt, ut = rows(p), rows(q) if drafts else None, torch.from_numpy(u).to(cuda_dev)
        e = torch.from_numpy(rng.exponential(size=(1, v)).astype(f)).to(cuda_dev).expand(b, v).contiguous()
        n, path, out = verify_tree(pt, tok, par, ut, e, qt)
        assert n[0] == 1 and n[-1] == 0                          # the sweep holds the edge
        for size in (1, 4, 9, 10):
            for at in range(0, b, size):
                part = slice(at, at + size)
                m, ph, o = verify_tree(pt[part], tok[part], par[part], ut[part], e[part], None if qt is None else qt[part])
                assert torch.equal(m, n[part]) and torch.equal(ph, path[part]) and torch.equal(o, out[part]), (seed, size, at)
