"""tree_attention_int8 at every height of a block of query rows (16, 32, 64 and several blocks of 64), with many tiles in a
block's range, ranges cut between blocks, and references that move from tile to tile; against torch in 64 bits.

Tolerances, per element, as for the trees of few tiles: u |o| + 2^-25 for the output's rounding (u = 2^-11 fp16, 2^-8
bf16), 2 (D + 4) 2^-24 reach for the scores' (reach: the largest scale * sum |q| |k| of a visible key), 2^-16 for the
exponential and the split of a weight, n 2^-24 for sums over n keys, the last three times a = sum w |v| / sum w."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}

ROWS = [  # t, hq, h: query rows of a key head
    (4, 16, 4), (16, 2, 2),                         # 16
    (17, 2, 2), (5, 7, 2), (6, 16, 4), (8, 16, 4), (31, 2, 2), (32, 1, 1),  # 17 to 32
    (11, 9, 3), (10, 16, 4), (16, 16, 4), (64, 2, 2),                       # 33 to 64
    (24, 8, 2), (64, 8, 2),                         # 96, 256: several blocks
]
ROWS = [(t, hq if hq % h == 0 else hq * h, h) for t, hq, h in ROWS]


def _cache(g, dev, b, h, d, page, slots):
    from blackwell_ops.decode import KVCacheInt8

    cols = -(-slots // page)
    pages = b * cols + 1
    k, v = (torch.randn((pages, h, page, d), generator=g, device=dev).mul_(32).round_().clamp_(-127, 127).to(torch.int8) for _ in "kv")
    ks, vs = ((torch.rand((pages, h, page), generator=g, device=dev) + 0.5) / 32 for _ in "kv")
    table = torch.randperm(pages, generator=g, device=dev)[: b * cols].to(torch.int32).view(b, cols)
    return KVCacheInt8(k, v, ks, vs), table


def _mask(g, dev, b, t):
    """Random visible nodes; node 0 of each sequence sees the context alone."""
    bits = torch.randint(0, 2, (b, t, t), generator=g, device=dev, dtype=torch.int64)
    bits[:, 0] = 0
    return (bits << torch.arange(t, device=dev)).sum(-1)


def _check(out, q, cache, table, ctx, mask, dt):
    b, t, hq, d = q.shape
    h, page = cache.heads, cache.page
    dev = q.device
    for i in range(b):
        n = int(ctx[i]) + t
        pg = table[i].long()
        k, v = ((c[pg].double() * s[pg].double()[..., None]).transpose(1, 2).reshape(-1, h, d)[:n]
                for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
        tree = ((mask[i][:, None] >> torch.arange(t, device=dev)) & 1) != 0
        see = torch.cat([tree.new_ones((t, n - t)), tree], 1)
        for x in range(hq):
            kk, vv, qq = k[:, x // (hq // h)], v[:, x // (hq // h)], q[i, :, x].double()
            s = (qq @ kk.T * d**-0.5).masked_fill(~see, -torch.inf)
            w = torch.softmax(s, -1)
            w = torch.where(see.any(-1, keepdim=True), w, 0)  # (no context, no node: zeros)
            o, a = w @ vv, w @ vv.abs()
            reach = float((qq.abs() @ kk.abs().T).masked_fill(~see, 0).max()) * d**-0.5
            err = (out[i, :, x].double() - o).abs()
            bound = U[dt] * o.abs() + 2.0**-25 + (2 * (d + 4) * 2.0**-24 * reach + 2.0**-16 + n * 2.0**-24) * a
            assert bool((err <= bound).all()), (i, x, float((err - bound).max()))


def _lens(b, top):
    return [top - (top // 2) * i // b for i in range(b)]


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 64)])
@pytest.mark.parametrize("t,hq,h", ROWS)
def test_heights(cuda_dev, t, hq, h, d, page, dt):
    """Short contexts (one or two tiles, some empty), one long one cut over many blocks, and a batch whose blocks hold
    many tiles each."""
    from blackwell_ops.decode import tree_attention_int8

    g = torch.Generator(device=cuda_dev).manual_seed(t * 100 + hq)
    for lens in ([0, 1, 127, 130], [9001], _lens(40, 2600)):
        b = len(lens)
        cache, table = _cache(g, cuda_dev, b, h, d, page, max(lens) + t)
        q = (2 * torch.randn((b, t, hq, d), generator=g, device=cuda_dev)).to(dt)
        mask = _mask(g, cuda_dev, b, t)
        ctx = torch.tensor(lens, dtype=torch.int32, device=cuda_dev)
        out = tree_attention_int8(q, cache, table, ctx, mask)
        some = list(range(0, b, max(1, b // 6)))
        _check(out[some], q[some], cache, table[some], ctx[some], mask[some], dt)
        if lens[0] == 0:
            assert not bool(out[0, 0].any())  # sees nothing
        assert torch.equal(out, tree_attention_int8(q, cache, table, ctx, mask)), "two runs differ"


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,page", [(64, 64), (128, 16)])
@pytest.mark.parametrize("t,hq,h", [(4, 16, 4), (8, 16, 4), (31, 2, 2), (16, 16, 4), (24, 8, 2)])
def test_moving_references(cuda_dev, t, hq, h, d, page, dt):
    """Scores that rise along the context, by up to 14 powers of two a tile and by another amount for each row, or fall:
    maxima move at different tiles in different rows, in blocks that hold several tiles and in cut ones.  Queries of
    one sign and positive codes: a score is its own sum of magnitudes, so reach is the largest score, about 110."""
    from blackwell_ops.decode import tree_attention_int8

    g = torch.Generator(device=cuda_dev).manual_seed(t + d)
    lens = _lens(40, 1500)
    b = len(lens)
    cache, table = _cache(g, cuda_dev, b, h, d, page, max(lens) + t)
    cache.k.copy_(cache.k.abs().clamp(min=20))
    slope = torch.linspace(0.0, 1.0, table.shape[1] * page, device=cuda_dev).view(1, -1, 1, page).expand(b, -1, h, page)
    # mean code 40, d of them times 0.25 times d^-0.5: a row of factor 1 scores 10 d^0.5 ks
    cache.k_scale[table.long()] = slope * (75.0 / (10 * d**0.5)) * (0.9 + 0.2 * torch.rand((b, table.shape[1], h, page), generator=g, device=cuda_dev))
    factor = torch.linspace(-1.3, 1.3, t * hq, device=cuda_dev).view(1, t, hq, 1)
    factor = factor[:, :, torch.randperm(hq, generator=g, device=cuda_dev)]
    q = (factor * 0.25 * (0.8 + 0.4 * torch.rand((b, t, hq, d), generator=g, device=cuda_dev))).to(dt)
    mask = _mask(g, cuda_dev, b, t)
    ctx = torch.tensor(lens, dtype=torch.int32, device=cuda_dev)
    out = tree_attention_int8(q, cache, table, ctx, mask)
    some = [0, 7, 20, 39]
    _check(out[some], q[some], cache, table[some], ctx[some], mask[some], dt)
