"""GPU parity of norms of queries and keys with the rotation (and the cache's write) against the CPU oracle.

Tolerances.  A row's factor 1 / sqrt(mean + eps) is off by half of the sum's relative error (16 additions of a lane and
four between lanes at most, 2^-24 each: 6e-7) and two ulps of the reciprocal root (2.4e-7), the two products by 2^-24
each: under 1e-6 of the value in all, before the turn, which adds 1e-6 of the pair's length (see test_gpu_rotary_kv).
One rounding to the type on top: half an ulp.  A key's scale follows its largest element (2e-6 and the quotient's
2^-24); its code may differ by one where the quotient lies near a rounding midpoint."""
import numpy as np
import pytest

from oracle import decode as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_rotary_kv import LLAMA3, U, YARN, _cache, _host, _i32, _np, _pair_length, _randn, _same, _table  # noqa: E402


def _near(got, x, w, eps, pos, plan, freq, mag, interleaved, dt):
    y = ref.norm(_np(x), None if w is None else _np(w), eps)
    want = ref.rotate(y, pos, freq, mag, interleaved)
    err = np.abs(_np(got).astype(np.float64) - want)
    length = np.maximum(plan.magnitude, 1) * _pair_length(y, plan.rot_dim, interleaved)
    bound = U[dt] * (np.abs(want) + 2e-6 * length) + 2.0**-25 + 2e-6 * length
    assert (err <= bound).all(), float((err - bound).max())
    return want


SHAPES = [(1, 1, 1, 2, 2, None), (1, 16, 8, 128, 128, None), (17, 32, 8, 128, 64, LLAMA3), (5, 3, 1, 80, 80, YARN),
          (9, 4, 2, 96, 48, None), (3, 5, 5, 66, 34, None), (130, 12, 1, 64, 64, LLAMA3), (2, 2, 1, 256, 256, YARN),
          (7, 28, 4, 32, 16, None), (1000, 8, 4, 128, 128, None)]


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,hq,hk,d,rot,scaling", SHAPES)
def test_norm_rotary(cuda_dev, n, hq, hk, d, rot, scaling, interleaved, dt):
    from blackwell_ops.decode import norm_rotary, rotary, rotary_frequencies, rotary_plan

    q, k = 4 * _randn(n, (n, hq, d), dt, cuda_dev), _randn(n + 1, (n, hk, d), dt, cuda_dev) / 8
    wq, wk = _randn(5, (d,), dt, cuda_dev), 1 + _randn(6, (d,), dt, cuda_dev) / 4
    pos = torch.randint(0, 131072, (n,), generator=torch.Generator().manual_seed(7))
    plan = rotary_plan(rot, 10000.0, scaling, interleaved, cuda_dev)
    freq, mag = rotary_frequencies(rot, 10000.0, scaling)
    for eps, weights in ((1e-6, (wq, wk)), (0.01, (wq, None)), (1e-5, (None, wk))):
        got = norm_rotary(q, k, pos.to(cuda_dev), plan, *weights, eps=eps)
        for y, x, w in zip(got, (q, k), weights):
            assert y.dtype == dt and y.shape == x.shape and y.is_contiguous()
            _near(y, x, w, eps, pos.numpy(), plan, freq.numpy(), mag, interleaved, dt)
    p32 = pos.to(torch.int32).to(cuda_dev)
    for y, z in zip(norm_rotary(q, k, p32, plan), rotary(q, k, p32, plan)):
        assert torch.equal(y, z)  # without weights: the rotation, bit for bit


def test_strides_and_extremes(cuda_dev):
    from blackwell_ops.decode import norm_rotary, rotary_frequencies, rotary_plan

    plan, (freq, mag) = rotary_plan(64, device=cuda_dev), rotary_frequencies(64)
    qkv = _randn(1, (3, 7, 16, 128), torch.float16, cuda_dev)
    w = 1 + _randn(2, (256,), torch.float16, cuda_dev) / 4
    cases = [(qkv[:, :, :8], qkv[:, :, 8:12]), (qkv[:, :, :8].transpose(0, 1), qkv[:, :, 8:12].transpose(0, 1)),
             (qkv[:, :, 1:9, 3:123], qkv[:, :, 9:11, 3:123]),
             (qkv[:, :1, :8].expand(3, 7, 8, 128), qkv[:, :, 8:9].expand(3, 7, 4, 128)), (qkv[:, :, :, ::2], None)]
    for q, k in cases:
        pos = torch.randint(0, 5000, q.shape[:-2], generator=torch.Generator().manual_seed(2), dtype=torch.int32)
        ws = w[::2][:q.shape[-1]]  # a strided weight
        got = norm_rotary(q, k, pos.to(cuda_dev), plan, ws, ws)
        for y, x in zip(got, (q, k)):
            if x is not None:
                _near(y, x, ws, 1e-6, pos.numpy(), plan, freq.numpy(), mag, False, torch.float16)
    # rows of zeros, of the type's largest values, of subnormal ones, and rows with NaN or an infinity, whose
    # neighbours are as they were
    x = _randn(3, (1, 8, 128), torch.bfloat16, cuda_dev)
    pos = torch.zeros(1, dtype=torch.int32, device=cuda_dev)
    plain, _ = norm_rotary(x, None, pos, plan, w[:128].bfloat16())
    y = x.clone()
    y[0, 1], y[0, 2], y[0, 3, 5], y[0, 4, 7] = 0, 1e-30, float("nan"), float("inf")
    got, _ = norm_rotary(y, None, pos, plan, w[:128].bfloat16())
    assert torch.equal(got[0, [0, 5, 6, 7]], plain[0, [0, 5, 6, 7]])
    assert not bool(got[0, 1].any()) and bool((got[0, 2].abs() < 1e-25).all())
    assert bool(got[0, 3].isnan().all()) and bool(got[0, 4, 7].isnan())
    h = torch.full((1, 1, 128), 65504.0, dtype=torch.float16, device=cuda_dev)  # its squares' sum is 5.5e11
    got, _ = norm_rotary(h, None, pos, plan, w[:128])
    _near(got, h, w[:128], 1e-6, np.zeros(1), plan, freq.numpy(), mag, False, torch.float16)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("b,t,hq,h,d,rot,page", [(1, 1, 4, 2, 128, 128, 16), (64, 1, 16, 8, 128, 128, 16), (3, 50, 8, 8, 64, 32, 64),
                                                 (2, 33, 3, 1, 80, 40, 7), (4, 17, 12, 1, 256, 256, 32), (2, 300, 28, 4, 128, 128, 5)])
def test_norm_write(cuda_dev, b, t, hq, h, d, rot, page, packed, interleaved, dt):
    from blackwell_ops.decode import norm_rotary, norm_rotary_kv_write_int8, rotary_frequencies, rotary_plan

    rng = np.random.default_rng(b * 1000 + t)
    start = rng.integers(0, 40, b).astype(np.int32)
    start[-1] = -3                          # slots that do not exist
    cols = int(40 + t + page - 1) // page
    cache, table = _cache(1, b * cols + 1, h, page, d, cuda_dev), _table(2, b, cols, b * cols + 1, cuda_dev)
    table[0, -1] = b * cols + 7             # no page
    lens = [t] * b if not packed else [max(0, t - 9 * i) if i != 1 else 0 for i in range(b)]  # (an empty one)
    off = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32) + (2 if packed else 0)
    n = int(off[-1]) + (5 if packed else 0)                                 # rows before the first and behind the last
    lead = (n,) if packed else (b, t)
    qkv = 2 * _randn(3, (*lead, hq + 2 * h, d), dt, cuda_dev)
    q, k, v = qkv.split([hq, h, h], dim=-2)
    wq, wk = 1 + _randn(5, (d,), dt, cuda_dev) / 4, 1 + _randn(6, (d,), dt, cuda_dev) / 4
    plan, (freq, mag) = rotary_plan(rot, 10000.0, LLAMA3, interleaved, cuda_dev), rotary_frequencies(rot, 10000.0, LLAMA3)
    pos = torch.randint(0, 100000, lead, generator=torch.Generator().manual_seed(3))
    before, tb = _host(cache), table.cpu().numpy()
    counts = None if packed else [max(0, t - i) for i in range(b)]
    got = norm_rotary_kv_write_int8(q, k, v, pos.to(cuda_dev), plan, cache, table, _i32(start, cuda_dev), wq, wk, eps=1e-5,
                                    counts=None if packed else _i32(counts, cuda_dev),
                                    offsets=_i32(off, cuda_dev) if packed else None, keys=True)
    for y, z in zip(got, norm_rotary(q, k, pos.to(cuda_dev), plan, wq, wk, eps=1e-5)):
        assert torch.equal(y, z)
    turned = _near(got[1], k, wk, 1e-5, pos.numpy(), plan, freq.numpy(), mag, interleaved, dt)
    want = [x.copy() for x in before]
    for i in range(b):
        rows = slice(off[i], off[i + 1]) if packed else i
        m = lens[i] if packed else counts[i]
        if m:
            ref.write(want, tb[i:i + 1], start[i:i + 1], turned[rows][None, :m], _np(v)[rows][None, :m])
    now = _host(cache)
    assert np.array_equal(now[1], want[1]) and np.array_equal(now[3], want[3])
    assert np.abs(now[2] / want[2] - 1).max() <= 2.2e-6
    diff = now[0].astype(int) - want[0].astype(int)
    assert np.abs(diff).max() <= 1 and (diff != 0).mean() <= 1e-3
    # the same without the keys, and without weights the rotation's write bit for bit
    again = _cache(1, b * cols + 1, h, page, d, cuda_dev)
    q2, none = norm_rotary_kv_write_int8(q, k, v, pos.to(cuda_dev), plan, again, table, _i32(start, cuda_dev), wq, wk, eps=1e-5,
                                         counts=None if packed else _i32(counts, cuda_dev),
                                         offsets=_i32(off, cuda_dev) if packed else None)
    assert none is None and torch.equal(q2, got[0])
    _same(again, now)
    if not packed:
        from blackwell_ops.decode import rotary_kv_write_int8

        one, two = (_cache(1, b * cols + 1, h, page, d, cuda_dev) for _ in "ab")
        args = (table, _i32(start, cuda_dev))
        y, _ = norm_rotary_kv_write_int8(q, k, v, pos.to(cuda_dev), plan, one, *args, counts=_i32(counts, cuda_dev))
        z = rotary_kv_write_int8(q, k, v, pos.to(cuda_dev), plan, two, *args, _i32(counts, cuda_dev))
        assert torch.equal(y, z)
        _same(one, _host(two))


def test_streams_and_graphs(cuda_dev):
    """Captured once and replayed on other inputs, on another stream than it was captured on."""
    from blackwell_ops.decode import norm_rotary_kv_write_int8, rotary_plan

    plan = rotary_plan(128, device=cuda_dev)
    w = torch.ones(128, dtype=torch.bfloat16, device=cuda_dev)
    x = _randn(1, (40, 4, 128), torch.bfloat16, cuda_dev)
    pos = torch.arange(40, dtype=torch.int32, device=cuda_dev)
    off, start = _i32([0, 11, 40], cuda_dev), _i32([0, 5], cuda_dev)
    cache, table = _cache(1, 9, 4, 16, 128, cuda_dev), _table(2, 2, 4, 9, cuda_dev)
    call = lambda c: norm_rotary_kv_write_int8(x, x, x, pos, plan, c, table, start, w, w, offsets=off, keys=True)  # noqa: E731
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call(cache)
    x.copy_(_randn(9, (40, 4, 128), torch.bfloat16, cuda_dev))
    off.copy_(_i32([0, 25, 37], cuda_dev))
    st = torch.cuda.Stream(cuda_dev)
    st.wait_stream(torch.cuda.current_stream(cuda_dev))
    with torch.cuda.stream(st):
        g.replay()
    torch.cuda.current_stream(cuda_dev).wait_stream(st)
    other = _cache(1, 9, 4, 16, 128, cuda_dev)
    want = call(other)
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    _same(cache, _host(other))


def test_offsets_out_of_order_stay_inside(cuda_dev):
    """Offsets that descend or pass the rows: what is written is undefined, but lies in the sequences' slots."""
    from blackwell_ops.decode import norm_rotary_kv_write_int8, rotary_plan

    plan = rotary_plan(64, device=cuda_dev)
    x = _randn(1, (30, 2, 64), torch.float16, cuda_dev)
    pos = torch.arange(30, dtype=torch.int32, device=cuda_dev)
    for off in ([0, 20, 10, 30], [5, 500, 1000, 2000], [-7, 3, -100, 12], [9, 8, 7, 6]):
        cache = _cache(1, 8, 2, 16, 64, cuda_dev)
        before = _host(cache)
        table = _i32([[0, 1], [2, 3], [4, 5]], cuda_dev)
        norm_rotary_kv_write_int8(x, x, x, pos, plan, cache, table, _i32([0, 0, 0], cuda_dev), offsets=_i32(off, cuda_dev))
        assert all(np.array_equal(a[6:], b[6:]) for a, b in zip(_host(cache), before))


def test_refusals(cuda_dev):
    from blackwell_ops import decode as D

    plan = D.rotary_plan(64, device=cuda_dev)
    x = torch.zeros((2, 3, 4, 64), dtype=torch.float16, device=cuda_dev)
    pos = torch.zeros((2, 3), dtype=torch.int32, device=cuda_dev)
    w = torch.ones(64, dtype=torch.float16, device=cuda_dev)
    cache = D.KVCacheInt8.empty(4, 4, 16, 64, device=cuda_dev)
    layered = D.KVCacheInt8.empty(4, 4, 16, 64, layers=2, device=cuda_dev)
    table, start, off = _i32([[0], [1]], cuda_dev), _i32([0, 0], cuda_dev), _i32([0, 1, 3], cuda_dev)
    write = D.norm_rotary_kv_write_int8
    for match, fn in [
        ("q must be CUDA", lambda: D.norm_rotary(x.cpu(), None, pos, plan)),
        ("fp16 or bf16", lambda: D.norm_rotary(x.float(), None, pos, plan)),
        ("leading dimensions", lambda: D.norm_rotary(x, x[:1], pos, plan)),
        ("q's dtype", lambda: D.norm_rotary(x, x.bfloat16(), pos, plan)),
        ("rot_dim", lambda: D.norm_rotary(x[..., :32], None, pos, plan)),
        ("q_weight must be", lambda: D.norm_rotary(x, None, pos, plan, w[:32])),
        ("q_weight must be", lambda: D.norm_rotary(x, None, pos, plan, w.float())),
        ("k_weight must be", lambda: D.norm_rotary(x, x, pos, plan, w, w.cpu())),
        ("eps must not", lambda: D.norm_rotary(x, x, pos, plan, w, w, eps=-1.0)),
        ("eps must not", lambda: D.norm_rotary(x, x, pos, plan, w, w, eps=float("nan"))),
        ("one layer", lambda: write(x, x, x, pos, plan, layered, table, start)),
        (r"\[B, T, heads, D\]", lambda: write(x[0], x[0], x[0], pos[0], plan, cache, table, start)),
        ("with offsets", lambda: write(x, x, x, pos, plan, cache, table, start, offsets=off)),
        ("no counts", lambda: write(x[0], x[0], x[0], pos[0], plan, cache, table, start, counts=start, offsets=off)),
        ("offsets must be", lambda: write(x[0], x[0], x[0], pos[0], plan, cache, table, start, offsets=start)),
        ("offsets must be int32", lambda: write(x[0], x[0], x[0], pos[0], plan, cache, table, start, offsets=off.long())),
        ("like the cache", lambda: write(x, x[:, :, :2], x[:, :, :2], pos, plan, cache, table, start)),
        ("one dtype", lambda: write(x, x, x.bfloat16(), pos, plan, cache, table, start)),
        ("a row for each", lambda: write(x, x, x, pos, plan, cache, table[:1], start)),
        ("start must be", lambda: write(x, x, x, pos, plan, cache, table, start[:1])),
        ("eps must not", lambda: write(x, x, x, pos, plan, cache, table, start, eps=-1.0)),
    ]:
        with pytest.raises(RuntimeError, match=match):
            fn()
    # empty problems
    y, none = D.norm_rotary(x[:0], None, pos[:0], plan, w)
    assert y.shape == (0, 3, 4, 64) and none is None
    write(x[:0], x[:0], x[:0], pos[:0], plan, cache, table[:0], start[:0], w, w)
    write(x[0, :0], x[0, :0], x[0, :0], pos[0, :0], plan, cache, table, start, w, w, offsets=_i32([0, 0, 0], cuda_dev))
    write(x[0], x[0], x[0], pos[0], plan, cache, table[:0], start[:0], w, w, offsets=_i32([0], cuda_dev))
    assert not bool(cache.k.any())
