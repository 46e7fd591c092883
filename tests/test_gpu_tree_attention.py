"""GPU parity of tree_attention_int8 against the oracle's attention in 64 bits.

Tolerances, per element.  o = sum w v / sum w.  The output is rounded once: u |o| (u = 2^-11 fp16, 2^-8 bf16; 2^-25 for
fp16's subnormals).  Before that a score carries the rounding of a sum of D exact products in fp32 and of three scalings:
delta <= (D + 4) 2^-24 scale sum |q| |k|, which moves each weight and the normaliser by that much relative: 2 delta; the
exponential and the split of a weight into two 16-bit parts add 2^-16; the fp32 sums over n keys n 2^-24.  All of these
scale with a = sum w |v| / sum w.  Over all elements the roundings are independent, so the error's norm is at most u
times the output's (rounding alone gives u / sqrt 3), where the outputs are not small against a.
"""
import numpy as np
import pytest

from oracle import decode as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def _i32(v, dev):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device=dev)


def _parents(rng, b, t):
    return np.array([[-1] + [rng.integers(max(0, i - 6), i) for i in range(1, t)] for _ in range(b)], dtype=np.int32)


def _setup(seed, b, t, hq, h, d, page, ctx, dt, dev, spare=2, qscale=2.0):
    """A cache whose unused slots hold NaN scales, scattered pages, and q as a slice of a wider projection."""
    from blackwell_ops.decode import KVCacheInt8

    rng = np.random.default_rng(seed)
    cols = (max(ctx) + t + page - 1) // page
    pages = b * cols + spare
    table = rng.permutation(pages)[: b * cols].astype(np.int32).reshape(b, cols)
    k, v = (np.clip(np.rint(rng.standard_normal((pages, h, page, d)) * 32), -127, 127).astype(np.int8) for _ in "kv")
    ks, vs = (np.full((pages, h, page), np.nan, dtype=np.float32) for _ in "kv")
    for i in range(b):
        for s in range(ctx[i] + t):
            pg, rw = table[i, s // page], s % page
            ks[pg, :, rw] = (rng.random(h) + 0.5) / 32
            vs[pg, :, rw] = (rng.random(h) + 0.5) / 32
    cache = KVCacheInt8(*(torch.from_numpy(x).to(dev) for x in (k, v, ks, vs)))
    q = torch.from_numpy(rng.standard_normal((b, t, hq + 2 * h, d)) * qscale).to(dt).to(dev)[:, :, :hq]
    return cache, [k, v, ks, vs], table, q, rng


def _check(out, q, host, table, ctx, dt, mask=None, counts=None, scale=None, norm=True):
    with np.errstate(invalid="ignore"):
        o, a, reach = ref.attention(q.float().cpu().numpy(), host, table, ctx, mask, counts, scale)
    d, n = q.shape[-1], max(ctx) + q.shape[1]
    delta = (d + 4) * 2.0**-24 * reach
    got = out.float().cpu().numpy().astype(np.float64)
    assert np.isfinite(got).all()
    err = np.abs(got - o)
    bound = U[dt] * np.abs(o) + 2.0**-25 + (2 * delta + 2.0**-16 + n * 2.0**-24) * a
    assert (err <= bound).all(), (float((err - bound).max()), np.argwhere(err > bound)[:4].tolist())
    if norm:
        assert np.linalg.norm(err) <= U[dt] * np.linalg.norm(o), np.linalg.norm(err) / np.linalg.norm(o)


CASES = [  # b, t, hq, h, d, page, ctx
    (1, 1, 1, 1, 64, 16, [0]), (1, 1, 16, 8, 128, 16, [1]), (2, 1, 8, 8, 128, 16, [127, 128]),
    (3, 1, 32, 8, 128, 64, [129, 5, 1000]), (2, 1, 12, 1, 64, 32, [300, 255]), (1, 2, 28, 4, 128, 16, [126]),
    (2, 5, 16, 8, 128, 16, [123, 700]), (1, 16, 32, 8, 128, 64, [513]), (2, 24, 32, 8, 64, 64, [10, 250]),
    (1, 33, 12, 1, 128, 128, [400]), (1, 64, 8, 8, 128, 16, [65]), (1, 64, 64, 8, 128, 64, [190]),
    (4, 64, 2, 1, 64, 128, [0, 1, 63, 200]), (2, 3, 4, 2, 80, 16, [77, 12]), (1, 7, 6, 2, 96, 32, [33]),
    (2, 2, 4, 4, 256, 16, [40, 9]), (2, 4, 3, 3, 33, 5, [50, 11]), (1, 5, 4, 4, 128, 7, [200]),
    (1, 1, 8, 8, 128, 256, [600]), (9, 1, 4, 1, 128, 16, [0, 1, 2, 15, 16, 17, 31, 511, 90]), (1, 1, 2, 1, 64, 16, [6000]),
]


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("b,t,hq,h,d,page,ctx", CASES)
def test_trees(cuda_dev, b, t, hq, h, d, page, ctx, dt):
    from blackwell_ops.decode import tree_attention_int8, tree_positions

    cache, host, table, q, rng = _setup(b * 1000 + t, b, t, hq, h, d, page, ctx, dt, cuda_dev)
    par = _parents(rng, b, t)
    mask, _ = tree_positions(_i32(par, cuda_dev))
    tb, c = _i32(table, cuda_dev), _i32(ctx, cuda_dev)
    out = tree_attention_int8(q, cache, tb, c, mask)
    assert out.dtype == dt and out.shape == q.shape
    _check(out, q, host, table, ctx, dt, ref.tree_mask(par)[0])
    assert torch.equal(out, tree_attention_int8(q, cache, tb, c, mask)), "two runs differ"
    _check(tree_attention_int8(q, cache, tb, c), q, host, table, ctx, dt)  # a chain


@pytest.mark.parametrize("d", [64, 128, 48])
def test_masks_that_hide(cuda_dev, d):
    """Nodes that see nothing, themselves only, later nodes, or nodes past a sequence's count; what nobody may see
    holds NaN and infinite scales."""
    from blackwell_ops.decode import KVCacheInt8, tree_attention_int8

    b, t, hq, h, page, ctx = 3, 9, 8, 2, 16, [0, 37, 128]
    dt = torch.float16
    cache, host, table, q, rng = _setup(5, b, t, hq, h, d, page, ctx, dt, cuda_dev)
    counts = [9, 6, 1]
    mask = rng.integers(0, 2**t, (b, t)).astype(np.uint64)
    mask[0, 0] = 0                       # sees nothing at all: no context either
    mask[0, 1] = np.uint64(1) << np.uint64(63)  # only a node that is not there
    mask[0, 2] = 1 << 8                  # a later node
    mask[1, 3] = 1 << 7                  # past the count: the context alone
    # node 4 of sequence 0 is seen by no one, node 5 by itself alone; their scales are not finite
    mask[0] &= ~np.uint64((1 << 4) | (1 << 5))
    mask[0, 5] = 1 << 8
    for node, val in ((4, np.inf), (5, np.nan)):
        pg, rw = table[0, node // page], node % page
        host[2][pg, :, rw] = host[3][pg, :, rw] = val
    for i, n in enumerate(counts):
        for s in range(ctx[i] + n, ctx[i] + t):  # never written
            host[2][table[i, s // page], :, s % page] = host[3][table[i, s // page], :, s % page] = np.inf
    cache = KVCacheInt8(*(torch.from_numpy(x).to(cuda_dev) for x in host))
    args = (cache, _i32(table, cuda_dev), _i32(ctx, cuda_dev), torch.from_numpy(mask.view(np.int64)).to(cuda_dev),
            _i32(counts, cuda_dev))
    out = tree_attention_int8(q, *args)
    _check(out, q, host, table, ctx, dt, mask, counts)
    assert not bool(out[0, 0].any()) and not bool(out[0, 1].any()) and not bool(out[1, 6:].any()) and not bool(out[2, 1:].any())
    # who does see such a node gets NaN, and no one else
    mask[0, 5] = (1 << 5) | 1
    out2 = tree_attention_int8(q, cache, args[1], args[2], torch.from_numpy(mask.view(np.int64)).to(cuda_dev), args[4])
    assert bool(out2[0, 5].isnan().all())
    keep = torch.ones_like(out[..., 0], dtype=torch.bool)
    keep[0, 5] = False
    assert torch.equal(out2[keep], out[keep])


@pytest.mark.parametrize("d,page", [(128, 16), (64, 64), (128, 12)])
def test_slots_that_do_not_exist(cuda_dev, d, page):
    """Lengths past the table, pages that are none of the cache's, negative lengths, shared prefix pages."""
    from blackwell_ops.decode import tree_attention_int8

    b, t, hq, h, ctx = 4, 3, 4, 2, [100, 100, 100, 90]
    dt = torch.bfloat16
    cache, host, table, q, _ = _setup(6, b, t, hq, h, d, page, ctx, dt, cuda_dev)
    table = table.copy()
    table[0, 1], table[1, 0] = -1, cache.pages
    table[3, :1] = table[2, :1]
    said = [103 + 50, 100, -7, 90]  # beyond the table; negative: no context
    out = tree_attention_int8(q, cache, _i32(table, cuda_dev), _i32(said, cuda_dev))
    # slots that exist but were never written hold NaN scales; sequence 0 sees some of them if its table has room
    room = table.shape[1] * page
    rows = [1, 2, 3] if room > 103 else [0, 1, 2, 3]
    _check(out[rows], q[rows], host, table[rows], [said[i] for i in rows], dt, norm=False)


def test_extreme_scores(cuda_dev):
    """Scores far from zero: one key takes all, and large equal ones; zero and tiny scales of values."""
    from blackwell_ops.decode import KVCacheInt8, tree_attention_int8

    for d in (64, 128):
        ctx, dt = [300], torch.float16
        cache, host, table, q, rng = _setup(8, 1, 4, 8, 2, d, 16, ctx, dt, cuda_dev, qscale=1.0)
        for j, (ks, vs) in {3: (40.0, 1.0), 250: (1e-30, 1e-30), 200: (0.0, 0.0), 17: (1 / 32, 1e-6), 30: (1 / 32, 200.0)}.items():
            pg, rw = table[0, j // 16], j % 16
            host[2][pg, :, rw], host[3][pg, :, rw] = ks, vs
        cache = KVCacheInt8(*(torch.from_numpy(x).to(cuda_dev) for x in host))
        out = tree_attention_int8(q, cache, _i32(table, cuda_dev), _i32(ctx, cuda_dev))
        o, _, _ = ref.attention(q.float().cpu().numpy(), host, table, ctx)
        # scores reach 1e4: their rounding moves weights; the key that takes all still gives its value to u
        assert np.linalg.norm(out.double().cpu().numpy() - o) <= 4e-3 * np.linalg.norm(o)
        # equal keys everywhere: the mean of the values, at scores of +-2000
        host[0][:] = 64
        host[2][np.isfinite(host[2])] = 1.0
        host[3][np.isfinite(host[3])] = 0.01
        cache = KVCacheInt8(*(torch.from_numpy(x).to(cuda_dev) for x in host))
        q2 = torch.full_like(q, 0.25)
        for sign in (1, -1):
            out = tree_attention_int8(q2 * sign, cache, _i32(table, cuda_dev), _i32(ctx, cuda_dev))
            _check(out, q2 * sign, host, table, ctx, dt)


@pytest.mark.parametrize("b,t,hq,h,d,page,ctx", [(2, 1, 8, 2, 128, 16, 5000), (1, 20, 8, 2, 64, 64, 4100), (1, 3, 2, 1, 128, 16, 20000)])
def test_long(cuda_dev, b, t, hq, h, d, page, ctx):
    """Long contexts split over many blocks, against torch in 64 bits on the GPU (the same bounds)."""
    from blackwell_ops.decode import tree_attention_int8

    ctx = [ctx - 777 * i for i in range(b)]
    dt = torch.float16
    cache, host, table, q, _ = _setup(9, b, t, hq, h, d, page, ctx, dt, cuda_dev)
    out = tree_attention_int8(q, cache, _i32(table, cuda_dev), _i32(ctx, cuda_dev))
    for i in range(b):
        n = ctx[i] + t
        pg = torch.from_numpy(table[i]).long().to(cuda_dev)
        k, v = ((c[pg].double() * s[pg].double()[..., None]).transpose(1, 2).reshape(-1, h, d)[:n]
                for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
        for x in range(hq):
            s = q[i, :, x].double() @ k[:, x // (hq // h)].T * d**-0.5
            see = torch.arange(n, device=cuda_dev) <= ctx[i] + torch.arange(t, device=cuda_dev)[:, None]
            w = torch.softmax(s.masked_fill(~see, -torch.inf), -1)
            vv = v[:, x // (hq // h)]
            o, a = w @ vv, w @ vv.abs()
            reach = float((q[i, :, x].double().abs() @ k[:, x // (hq // h)].abs().T).max()) * d**-0.5
            err = (out[i, :, x].double() - o).abs()
            bound = U[dt] * o.abs() + 2.0**-25 + (2 * (d + 4) * 2.0**-24 * reach + 2.0**-16 + n * 2.0**-24) * a
            assert bool((err <= bound).all()), float((err - bound).max())


@pytest.mark.parametrize("b,t,hq,h,d,page", [
    (700, 1, 4, 2, 64, 16),      # more sequences than one launch takes
    (2, 1, 12000, 1, 64, 16),    # more blocks of query rows than SMs
    (1, 3, 11200, 1, 64, 16),    # more query rows than the tickets cover
])
def test_many_sequences_and_heads(cuda_dev, b, t, hq, h, d, page):
    """Shapes at the ends of the grid, with calls of an ordinary shape on the same workspace between them."""
    from blackwell_ops.decode import tree_attention_int8

    dt = torch.float16
    small = _setup(21, 3, 2, 8, 2, 128, 16, [700, 40, 3000], dt, cuda_dev)
    args = (small[3], small[0], _i32(small[2], cuda_dev), _i32([700, 40, 3000], cuda_dev))
    before = tree_attention_int8(*args)
    _check(before, small[3], small[1], small[2], [700, 40, 3000], dt)
    rng = np.random.default_rng(22)
    ctx = [int(x) for x in rng.integers(0, 40, b)]
    cache, host, table, q, _ = _setup(23, b, t, hq, h, d, page, ctx, dt, cuda_dev)
    for _ in range(2):
        out = tree_attention_int8(q, cache, _i32(table, cuda_dev), _i32(ctx, cuda_dev))
        _check(out, q, host, table, ctx, dt)
        assert torch.equal(tree_attention_int8(*args), before)


def test_offsets_past_32_bits(cuda_dev):
    from blackwell_ops.decode import KVCacheInt8, tree_attention_int8

    pages, h, page, d = 33000, 8, 64, 128
    cache = KVCacheInt8(*(torch.empty((pages, h, page, d), dtype=torch.int8, device=cuda_dev) for _ in "kv"),
                        *(torch.full((pages, h, page), float("nan"), device=cuda_dev) for _ in "kv"))
    small, host, table, q, _ = _setup(10, 1, 2, 16, h, d, page, [250], torch.bfloat16, cuda_dev, spare=0)
    n = table.shape[1]
    far = torch.arange(pages - n, pages, device=cuda_dev)
    for x, y in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), (small.k, small.v, small.k_scale, small.v_scale)):
        x[far] = y[torch.from_numpy(table[0]).long().to(cuda_dev)]
    c = _i32([250], cuda_dev)
    a = tree_attention_int8(q, cache, far.to(torch.int32)[None], c)
    assert torch.equal(a, tree_attention_int8(q, small, _i32(table, cuda_dev), c))


def test_streams_strides_and_graph(cuda_dev):
    """The same outputs for another order of q's memory, on another stream, and replayed from a CUDA graph after the
    lengths have changed."""
    from blackwell_ops.decode import tree_attention_int8

    dt = torch.float16
    cache, host, table, q, _ = _setup(11, 2, 5, 16, 8, 128, 16, [300, 280], dt, cuda_dev)
    tb, c = _i32(table, cuda_dev), _i32([300, 41], cuda_dev)
    want = tree_attention_int8(q, cache, tb, c)
    assert torch.equal(want, tree_attention_int8(q.transpose(1, 2).contiguous().transpose(1, 2), cache, tb, c))
    wide = torch.cat([tb, tb.flip(1)], 1)[:, : tb.shape[1]]  # a table with a wider row
    assert torch.equal(want, tree_attention_int8(q.flip(3).flip(3), cache, wide, c))
    shifted = torch.empty(q.numel() + 1, dtype=dt, device=cuda_dev)[1:].view(q.shape).copy_(q)  # 2-byte alignment
    assert torch.equal(want, tree_attention_int8(shifted, cache, tb, c))
    st = torch.cuda.Stream(cuda_dev)
    st.wait_stream(torch.cuda.current_stream(cuda_dev))
    with torch.cuda.stream(st):
        other = tree_attention_int8(q, cache, tb, c)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            out = tree_attention_int8(q, cache, tb, c)
    st.synchronize()
    assert torch.equal(want, other)
    for lens in ([300, 41], [0, 280], [17, 3]):
        c.copy_(_i32(lens, cuda_dev))
        g.replay()
        torch.cuda.synchronize(cuda_dev)
        _check(out, q, host, table, lens, dt)


def test_refusals(cuda_dev):
    from blackwell_ops.decode import KVCacheInt8, tree_attention_int8

    cache = KVCacheInt8.empty(4, 2, 16, 64, device=cuda_dev)
    q = torch.zeros((2, 3, 4, 64), dtype=torch.float16, device=cuda_dev)
    table, ctx = _i32([[0], [1]], cuda_dev), _i32([4, 4], cuda_dev)
    for match, args, kw in [
        ("fp16 or bf16", (q.float(), cache, table, ctx), {}), ("fp16 or bf16", (q.cpu(), cache, table, ctx), {}),
        (r"\[B, T, heads, D\]", (q[0], cache, table, ctx), {}), ("head dimension", (q[..., :32], cache, table, ctx), {}),
        ("multiple", (q[:, :, :3], cache, table, ctx), {}), ("multiple", (q[:, :, :0], cache, table, ctx), {}),
        ("at most 64", (q[:, :1].expand(2, 65, 4, 64), cache, table, ctx), {}),
        ("table must be int32", (q, cache, table.long(), ctx), {}), ("a row for each", (q, cache, table[:1], ctx), {}),
        ("ctx_lens must be", (q, cache, table, ctx[:1]), {}), ("ctx_lens must be", (q, cache, table, None), {}),
        ("mask must be", (q, cache, table, ctx), dict(mask=ctx)), ("counts must be", (q, cache, table, ctx), dict(counts=ctx[:1])),
        ("one layer", (q, KVCacheInt8.empty(4, 2, 16, 64, layers=1, device=cuda_dev), table, ctx), {}),
    ]:
        with pytest.raises(RuntimeError, match=match):
            tree_attention_int8(*args, **kw)
    assert tree_attention_int8(q[:0], cache, table[:0], ctx[:0]).shape == (0, 3, 4, 64)
    assert tree_attention_int8(q[:, :0], cache, table, ctx).shape == (2, 0, 4, 64)
