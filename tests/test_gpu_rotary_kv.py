"""GPU parity of rotary positions and the paged int8 KV cache against the CPU oracle (oracle/decode.py).

Tolerances.  A rotated value is rounded once to its type: half an ulp (u = 2^-11 of it in fp16, 2^-8 in bf16), and
before that carries the 32-bit arithmetic's error: the angle is off by at most 2^-25 half turns (1e-7 radians) and each
of the sine, cosine, two products and the sum by 2^-23 at most, under 1e-6 of the pair's length in all; 2^-25 is fp16's
subnormal rounding.  Codes and scales of plain writes, of reads and of moves are exact.  A rotated key's scale follows
its largest element (1e-6), and its code may differ by one where the quotient lies near a rounding midpoint: read back
as values they differ by at most the step and 1e-6 of the row's length.
"""
import numpy as np
import pytest

from oracle import decode as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}
YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096}


def _randn(seed, shape, dt, dev):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dt).to(dev)


def _np(x):
    return x.detach().float().cpu().numpy() if x.is_floating_point() else x.detach().cpu().numpy()


def _pair_length(x, rot, interleaved):
    """The length of each element's pair (of itself where it does not turn)."""
    y = np.abs(x.astype(np.float64))
    half = rot // 2
    i, j = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, half), slice(half, rot))
    y[..., i] = y[..., j] = np.hypot(y[..., i], y[..., j])
    return y


def _near(got, want, x, plan, dt):
    err = np.abs(_np(got).astype(np.float64) - want)
    bound = U[dt] * np.abs(want) + 2.0**-25 + 1e-6 * plan.magnitude * _pair_length(_np(x), plan.rot_dim, plan.interleaved)
    assert (err <= bound).all(), float((err - bound).max())


def _cache(seed, pages, h, page, d, dev, layers=None):
    from blackwell_ops.decode import KVCacheInt8

    g = torch.Generator().manual_seed(seed)
    shape = (pages, h, page, d) if layers is None else (layers, pages, h, page, d)
    k, v = (torch.randint(-127, 128, shape, generator=g, dtype=torch.int8).to(dev) for _ in "kv")
    ks, vs = (((torch.rand(shape[:-1], generator=g) + 0.1) / 32).to(dev) for _ in "kv")
    return KVCacheInt8(k, v, ks, vs)


def _host(cache):
    return [x.cpu().numpy().copy() for x in (cache.k, cache.v, cache.k_scale, cache.v_scale)]


def _table(seed, b, cols, pages, dev):
    p = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[: b * cols]
    return p.to(torch.int32).view(b, cols).to(dev)


def _i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _same(cache, want):
    for name, x, w in zip(("k", "v", "k_scale", "v_scale"), (cache.k, cache.v, cache.k_scale, cache.v_scale), want):
        got = x.cpu().numpy()
        if got.dtype == np.float32:
            got, w = got.view(np.uint32), w.view(np.uint32)
        assert np.array_equal(got, w), f"{name}: {np.argwhere(got != w)[:4].tolist()}"


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,hq,hk,d,rot,scaling,top", [
    (1, 1, 1, 2, 2, None, 8), (1, 16, 8, 128, 128, None, 4096), (17, 32, 8, 128, 64, LLAMA3, 131072),
    (5, 3, 1, 80, 80, YARN, 16384), (9, 4, 2, 96, 48, None, 1 << 20), (3, 5, 5, 66, 34, None, 2**31 - 1),
    (130, 12, 1, 64, 64, LLAMA3, 131072), (2, 2, 1, 256, 256, YARN, 65536), (1000, 8, 4, 128, 128, None, 131072)])
def test_rotary(cuda_dev, n, hq, hk, d, rot, scaling, top, interleaved, dt):
    from blackwell_ops.decode import rotary, rotary_frequencies, rotary_plan

    q, k = _randn(n, (n, hq, d), dt, cuda_dev), _randn(n + 1, (n, hk, d), dt, cuda_dev)
    pos = torch.randint(0, top, (n,), generator=torch.Generator().manual_seed(7))
    pos[0] = top - 1
    plan = rotary_plan(rot, 10000.0, scaling, interleaved, cuda_dev)
    freq, mag = rotary_frequencies(rot, 10000.0, scaling)
    assert mag == plan.magnitude
    for p in (pos.to(torch.int32).to(cuda_dev), pos.to(cuda_dev)):
        for got, x in zip(rotary(q, k, p, plan), (q, k)):
            assert got.dtype == dt and got.shape == x.shape and got.is_contiguous()
            _near(got, ref.rotate(_np(x), pos.numpy(), freq.numpy(), mag, interleaved), x, plan, dt)


def test_rotary_strides_and_shapes(cuda_dev):
    from blackwell_ops.decode import rotary, rotary_frequencies, rotary_plan

    plan, (freq, mag) = rotary_plan(64, device=cuda_dev), rotary_frequencies(64)
    dt = torch.float16
    qkv = _randn(1, (3, 7, 16, 128), dt, cuda_dev)
    cases = [(qkv[:, :, :8], qkv[:, :, 8:12]),                                    # slices of one projection
             (qkv[:, :, :8].transpose(0, 1), qkv[:, :, 8:12].transpose(0, 1)),    # batch and time exchanged
             (qkv[:, :, 1:9, 3:123], qkv[:, :, 9:11, 3:123]),                     # unaligned starts, D = 120
             (qkv[:, :1, :8].expand(3, 7, 8, 128), qkv[:, :, 8:9].expand(3, 7, 4, 128)),  # broadcast tokens and heads
             (qkv[:, :, :, ::2], None),                                           # strided elements, no keys
             (qkv.transpose(1, 2), None)]                                         # heads and time exchanged
    for q, k in cases:
        pos = torch.randint(0, 5000, q.shape[:-2], generator=torch.Generator().manual_seed(2), dtype=torch.int32)
        got = rotary(q, k, pos.to(cuda_dev), plan)
        assert (got[1] is None) == (k is None)
        for y, x in zip(got, (q, k)):
            if x is not None:
                _near(y, ref.rotate(_np(x), pos.numpy(), freq.numpy(), mag), x, plan, dt)
    # positions in another order of memory, negative positions, five dimensions, nothing at all
    x = _randn(3, (2, 3, 4, 2, 64), dt, cuda_dev)
    pos = torch.arange(24, dtype=torch.int32).view(4, 3, 2).permute(2, 1, 0) - 12
    y, _ = rotary(x, None, pos.to(cuda_dev), plan)
    _near(y, ref.rotate(_np(x), pos.numpy(), freq.numpy(), mag), x, plan, dt)
    y, z = rotary(x[:0, 0], x[:0, 0], torch.empty((0, 4), dtype=torch.int32, device=cuda_dev), plan)
    assert y.shape == (0, 4, 2, 64) and z.shape == (0, 4, 2, 64)


def test_rotary_keeps_products(cuda_dev):
    """q . k depends on the difference of positions only, far out too (bf16 rounding: 64 products of O(1))."""
    from blackwell_ops.decode import rotary, rotary_plan

    plan = rotary_plan(64, 500000.0, device=cuda_dev)
    q, k = _randn(1, (1, 1, 64), torch.float16, cuda_dev), _randn(2, (1, 1, 64), torch.float16, cuda_dev)
    n = 64
    near = torch.arange(n, dtype=torch.int32, device=cuda_dev)
    dots = []
    for base in (0, 1_000_000_000):
        a, _ = rotary(q.expand(n, 1, 64), None, near + base + 100, plan)
        b, _ = rotary(k.expand(n, 1, 64), None, near + base, plan)
        dots.append((a.double() * b.double()).sum(-1))
    # each product of two roundings: 2 * 2^-11 * |q_i k_i|, and 64 of them
    tol = 2 * 2.0**-10 * float((q.double().norm() * k.double().norm()))
    assert float((dots[0] - dots[0][0]).abs().max()) <= tol and float((dots[1] - dots[0]).abs().max()) <= tol


SHAPES = [(1, 1, 1, 128, 16), (3, 5, 8, 128, 16), (2, 33, 2, 64, 64), (4, 2, 3, 80, 7), (2, 19, 1, 96, 32),
          (5, 1, 4, 256, 128), (2, 3, 2, 33, 5), (1, 300, 8, 128, 64)]


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("b,t,h,d,page", SHAPES)
def test_write_read_exact(cuda_dev, b, t, h, d, page, dt):
    from blackwell_ops.decode import kv_read_int8, kv_write_int8

    start = [(7 * i) % 23 for i in range(b)]
    cols = (max(start) + t + page - 1) // page
    pages = b * cols + 2
    cache, table = _cache(1, pages, h, page, d, cuda_dev), _table(2, b, cols, pages, cuda_dev)
    want = _host(cache)
    x = _randn(3, (b, t, h, d), dt, cuda_dev) * 3
    y = _randn(4, (b, h, t, d), dt, cuda_dev).transpose(1, 2)  # other strides for v
    counts = [t - (i % 2) * (t // 2) for i in range(b)]
    kv_write_int8(x, y, cache, table, _i32(start, cuda_dev), _i32(counts, cuda_dev))
    tb = table.cpu().numpy()
    ref.write(want, tb, start, _np(x), _np(y), counts)
    _same(cache, want)
    kv_write_int8(x, y, cache, table, _i32(start, cuda_dev))
    ref.write(want, tb, start, _np(x), _np(y))
    _same(cache, want)
    for st, n, lens in ((start, t, None), (None, cols * page + 3, None), (start, t + 2, [i % (t + 2) for i in range(b)])):
        got = kv_read_int8(cache, table, None if st is None else _i32(st, cuda_dev), n,
                           None if lens is None else _i32(lens, cuda_dev), dt)
        exact = ref.read(want, tb, st, n, lens)
        for g, e in zip(got, exact):
            assert g.dtype == dt and torch.equal(g.cpu(), torch.from_numpy(e).float().to(dt))


def test_write_edge_rows(cuda_dev):
    """Rows of zeros, NaN, infinities, subnormals and exact half-way quotients; slots that do not exist."""
    from blackwell_ops.decode import kv_read_int8, kv_write_int8

    for d in (128, 64, 40):
        x = _randn(1, (2, 8, 2, d), torch.float16, "cpu")
        x[0, 0] = 0
        x[0, 1, :, ::3] = float("nan")
        x[0, 2, 0, 5] = float("inf")
        x[0, 3] = float("nan")
        x[0, 4] = 6e-8
        x[0, 5] = 0
        x[0, 5, :, :9] = torch.tensor([127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 126.5, -126.5])
        x[0, 6, 1, 3] = -65504.0
        x[0, 7, 0, 7] = float("-inf")
        x = x.to(cuda_dev)
        cache = _cache(1, 6, 2, 4, d, cuda_dev)
        want = _host(cache)
        # sequence 1's second page is none of the cache's, its third is negative; the table ends after it
        table = _i32([[5, 0, 3], [1, 6, -1]], cuda_dev)
        start = [3, 1]
        kv_write_int8(x, x, cache, table, _i32(start, cuda_dev))
        ref.write(want, table.cpu().numpy(), start, _np(x), _np(x))
        for a, w in zip((cache.k, cache.v), want):
            assert np.array_equal(a.cpu().numpy(), w)
        assert np.array_equal(cache.k_scale.cpu().numpy(), want[2], equal_nan=True)
        k, _ = kv_read_int8(cache, table, _i32(start, cuda_dev), 8)
        with np.errstate(invalid="ignore"):
            e = ref.read(want, table.cpu().numpy(), start, 8)[0]
        assert torch.equal(torch.nan_to_num(k.cpu(), 7.0), torch.nan_to_num(torch.from_numpy(e).half(), 7.0))
        # a start before the first slot and one past every page write what exists
        kv_write_int8(x, x, cache, table, _i32([-3, 1000], cuda_dev))
        ref.write(want, table.cpu().numpy(), [-3, 1000], _np(x), _np(x))
        assert np.array_equal(cache.k.cpu().numpy(), want[0])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b,t,hq,h,d,rot,page,dt", [
    (1, 1, 16, 8, 128, 128, 16, torch.float16), (3, 9, 8, 2, 128, 64, 64, torch.bfloat16),
    (2, 5, 3, 3, 64, 64, 32, torch.bfloat16), (2, 4, 2, 1, 80, 40, 7, torch.float16),
    (1, 130, 12, 1, 256, 256, 128, torch.bfloat16), (2, 3, 0, 2, 64, 32, 16, torch.float16)])
def test_rotary_write(cuda_dev, b, t, hq, h, d, rot, page, dt, interleaved):
    from blackwell_ops.decode import rotary, rotary_frequencies, rotary_kv_write_int8, rotary_plan

    start = [11 * i + 2 for i in range(b)]
    cols = (max(start) + t + page - 1) // page
    cache, table = _cache(1, b * cols, h, page, d, cuda_dev), _table(2, b, cols, b * cols, cuda_dev)
    before = _host(cache)
    qkv = _randn(3, (b, t, hq + 2 * h, d), dt, cuda_dev)
    q, k, v = qkv.split([hq, h, h], dim=2)
    pos = torch.randint(0, 100000, (b, t), generator=torch.Generator().manual_seed(5), dtype=torch.int32)
    plan = rotary_plan(rot, 500000.0, YARN, interleaved, cuda_dev)
    freq, mag = rotary_frequencies(rot, 500000.0, YARN)
    counts = [t - i for i in range(b)]
    got = rotary_kv_write_int8(q, k, v, pos.to(cuda_dev), plan, cache, table, _i32(start, cuda_dev),
                               _i32(counts, cuda_dev))
    if hq:
        assert torch.equal(got, rotary(q, None, pos.to(cuda_dev), plan)[0])
    want = [x.copy() for x in before]
    turned = ref.rotate(_np(k), pos.numpy(), freq.numpy(), mag, interleaved)
    tb = table.cpu().numpy()
    ref.write(want, tb, start, turned, _np(v), counts)
    now = _host(cache)
    assert np.array_equal(now[1], want[1]) and np.array_equal(now[3], want[3])
    assert np.abs(now[2] / want[2] - 1).max() <= 2e-6
    off = now[0].astype(int) - want[0].astype(int)
    assert np.abs(off).max() <= 1 and (off != 0).mean() <= 1e-3
    x = ref.read(now, tb, start, t, counts)[0]
    length = np.linalg.norm(turned, axis=-1, keepdims=True)
    for i in range(b):
        n = counts[i]
        step = np.abs(turned[i, :n]).max(-1, keepdims=True) / 127
        assert (np.abs(x[i, :n] - turned[i, :n]) <= 0.5 * step * (1 + 1e-4) + 2e-6 * length[i, :n]).all()


@pytest.mark.parametrize("layers,b,t,h,d,page", [(None, 1, 2, 1, 64, 16), (3, 4, 16, 2, 128, 16), (2, 3, 64, 8, 128, 64),
                                                 (2, 5, 9, 3, 80, 5), (1, 2, 33, 2, 33, 7), (2, 1, 64, 1, 256, 128)])
def test_move(cuda_dev, layers, b, t, h, d, page):
    from blackwell_ops.decode import kv_move_int8, kv_read_int8

    rng = np.random.default_rng(t * 100 + b)
    start = rng.integers(0, 40, b)
    cols = int(start.max() + t + page - 1) // page
    cache, table = _cache(1, b * cols + 1, h, page, d, cuda_dev, layers), _table(2, b, cols, b * cols + 1, cuda_dev)
    taken = rng.integers(0, t, b)
    taken[0] = t - 1
    path = np.full((b, t), -1, dtype=np.int32)
    for i in range(b):  # ascending paths that overlap their targets, and one in any order
        path[i, : taken[i]] = np.sort(rng.choice(np.arange(1, t), taken[i], replace=False))
    if b > 2:
        path[2, : taken[2]] = rng.permutation(path[2, : taken[2]])
    if b > 3:
        path[3, 0] = t + 5  # no node
    want = _host(cache)
    kv_move_int8(cache, table, _i32(start, cuda_dev), _i32(path, cuda_dev), _i32(taken, cuda_dev))
    tb = table.cpu().numpy()
    if layers is None:
        ref.move(want, tb, start, path, taken)
    else:
        for i in range(layers):
            ref.move([x[i] for x in want], tb, start, path, taken)
    _same(cache, want)
    k, v = kv_read_int8(cache, table, _i32(start, cuda_dev), t, dtype=torch.bfloat16)
    for i in range(layers or 0):
        kk, vv = kv_read_int8(cache.layer(i), table, _i32(start, cuda_dev), t, dtype=torch.bfloat16)
        assert torch.equal(k[i], kk) and torch.equal(v[i], vv)


def test_offsets_past_32_bits(cuda_dev):
    """A cache of more than 2^31 codes: written, moved and read at its end."""
    from blackwell_ops.decode import KVCacheInt8, kv_move_int8, kv_read_int8, kv_write_int8

    pages, h, page, d = 33000, 8, 64, 128
    assert pages * h * page * d > 2**31
    cache = KVCacheInt8(*(torch.empty((pages, h, page, d), dtype=torch.int8, device=cuda_dev) for _ in "kv"),
                        *(torch.empty((pages, h, page), device=cuda_dev) for _ in "kv"))
    table = _i32([[pages - 1, 0, pages - 2]], cuda_dev)
    x = _randn(1, (1, 150, h, d), torch.float16, cuda_dev)
    kv_write_int8(x, -x, cache, table, _i32([10], cuda_dev))
    codes, s = ref.quantise(_np(x))
    want = torch.from_numpy(codes.astype(np.float32) * s[..., None]).half()
    k, v = kv_read_int8(cache, table, _i32([10], cuda_dev), 150)
    assert torch.equal(k.cpu(), want) and torch.equal(v.cpu(), -want)
    kv_move_int8(cache, table, _i32([130], cuda_dev), _i32([[20, 25, -1] + [-1] * 29], cuda_dev), _i32([2], cuda_dev))
    k, _ = kv_read_int8(cache, table, _i32([131], cuda_dev), 2)
    assert torch.equal(k.cpu()[0], want[0, [140, 145]])


def test_tree_positions(cuda_dev):
    from blackwell_ops.decode import tree_positions

    rng = np.random.default_rng(3)
    for t in (1, 2, 7, 32, 64):
        par = np.array([[-1] + [rng.integers(0, i) for i in range(1, t)] for _ in range(9)], dtype=np.int32)
        par[1] = np.arange(t) - 1
        if t > 4:
            par[2, 3:] = -1                     # padding
            par[3, 2], par[4, 2] = 2, t + 3     # its own parent; a later node
        ctx = rng.integers(0, 1 << 20, 9).astype(np.int32)
        mask, depth = ref.tree_mask(par)
        m, p = tree_positions(_i32(par, cuda_dev), _i32(ctx, cuda_dev))
        assert np.array_equal(m.cpu().numpy().view(np.uint64), mask)
        assert np.array_equal(p.cpu().numpy(), depth + ctx[:, None])
        assert np.array_equal(tree_positions(_i32(par, cuda_dev))[1].cpu().numpy(), depth)


def test_side_stream(cuda_dev):
    """Inputs made, written and read on another stream than the default one."""
    from blackwell_ops.decode import kv_read_int8, kv_write_int8, rotary, rotary_plan

    plan = rotary_plan(128, device=cuda_dev)
    cache, table = _cache(1, 70, 8, 16, 128, cuda_dev), _table(2, 1, 70, 70, cuda_dev)
    st = torch.cuda.Stream(cuda_dev)
    st.wait_stream(torch.cuda.current_stream(cuda_dev))
    with torch.cuda.stream(st):
        x = torch.zeros((1, 1024, 8, 128), dtype=torch.float16, device=cuda_dev)
        for _ in range(50):
            x += 1
        kv_write_int8(x, x, cache, table, _i32([0], cuda_dev))
        k, _ = kv_read_int8(cache, table, None, 1024)
        y, _ = rotary(x, None, torch.zeros((1, 1024), dtype=torch.int32, device=cuda_dev), plan)
    st.synchronize()
    assert torch.equal(y, x) and bool((k == 50).all())


def test_refusals(cuda_dev):
    from blackwell_ops import decode as D

    plan = D.rotary_plan(64, device=cuda_dev)
    x = torch.zeros((2, 3, 4, 64), dtype=torch.float16, device=cuda_dev)
    pos = torch.zeros((2, 3), dtype=torch.int32, device=cuda_dev)
    cache = D.KVCacheInt8.empty(4, 4, 16, 64, device=cuda_dev)
    layered = D.KVCacheInt8.empty(4, 4, 16, 64, layers=2, device=cuda_dev)
    table, start = _i32([[0], [1]], cuda_dev), _i32([0, 0], cuda_dev)
    for match, fn in [
        ("q must be CUDA", lambda: D.rotary(x.cpu(), None, pos, plan)),
        ("fp16 or bf16", lambda: D.rotary(x.float(), None, pos, plan)),
        (r"\[\.\., heads, d\]", lambda: D.rotary(x[0, 0], None, pos, plan)),
        ("leading dimensions", lambda: D.rotary(x, x[:1], pos, plan)),
        ("q's dtype", lambda: D.rotary(x, x.bfloat16(), pos, plan)),
        ("positions must be", lambda: D.rotary(x, None, pos[:1], plan)),
        ("int32 or int64", lambda: D.rotary(x, None, pos.float(), plan)),
        ("rot_dim", lambda: D.rotary(x[..., :32], None, pos, plan)),
        ("even", lambda: D.rotary_plan(63, device=cuda_dev)),
        ("unknown scaling", lambda: D.rotary_plan(64, scaling={"rope_type": "other", "factor": 2.0}, device=cuda_dev)),
        ("needs factor", lambda: D.rotary_plan(64, scaling={"rope_type": "linear"}, device=cuda_dev)),
        ("must be positive", lambda: D.rotary_plan(64, scaling={"rope_type": "linear", "factor": 0}, device=cuda_dev)),
        ("codes must be int8", lambda: D.KVCacheInt8(cache.k.half(), cache.v, cache.k_scale, cache.v_scale)),
        ("scales must be fp32", lambda: D.KVCacheInt8(cache.k, cache.v, cache.k_scale.half(), cache.v_scale)),
        ("same layers", lambda: D.KVCacheInt8(cache.k, cache.v[:2], cache.k_scale, cache.v_scale)),
        ("contiguous", lambda: D.KVCacheInt8(*(t.transpose(0, 1) for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)))),
        ("head dimension must be", lambda: D.KVCacheInt8.empty(1, 1, 1, 264, device=cuda_dev)),
        ("one layer", lambda: D.kv_write_int8(x, x, layered, table, start)),
        ("like the cache", lambda: D.kv_write_int8(x[:, :, :2], x[:, :, :2], cache, table, start)),
        ("one dtype", lambda: D.kv_write_int8(x, x.bfloat16(), cache, table, start)),
        ("table must be int32", lambda: D.kv_write_int8(x, x, cache, table.long(), start)),
        ("a row for each", lambda: D.kv_write_int8(x, x, cache, table[:1], start)),
        ("start must be", lambda: D.kv_write_int8(x, x, cache, table, start[:1])),
        ("start must be", lambda: D.kv_write_int8(x, x, cache, table, None)),
        ("counts must be int32", lambda: D.kv_write_int8(x, x, cache, table, start, start.long())),
        ("fp16 or bf16", lambda: D.kv_read_int8(cache, table, None, 4, dtype=torch.float32)),
        ("negative", lambda: D.kv_read_int8(cache, table, None, -1)),
        ("path must be", lambda: D.kv_move_int8(cache, table, start, torch.zeros((2, 65), dtype=torch.int32, device=cuda_dev), start)),
        ("taken must be", lambda: D.kv_move_int8(cache, table, start, torch.zeros((2, 4), dtype=torch.int32, device=cuda_dev), None)),
        ("parents must be", lambda: D.tree_positions(torch.zeros((2, 65), dtype=torch.int32, device=cuda_dev))),
        ("no layers", lambda: cache.layer(0)),
    ]:
        with pytest.raises(RuntimeError, match=match):
            fn()
    # empty problems
    D.kv_write_int8(x[:0], x[:0], cache, table[:0], start[:0])
    D.kv_write_int8(x[:, :0], x[:, :0], cache, table, start)
    assert D.kv_read_int8(cache, table, None, 0)[0].shape == (2, 0, 4, 64)
    assert not bool(cache.k.any())
