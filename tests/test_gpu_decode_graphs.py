"""Captured attention calls: what a graph replays does not depend on what runs, grows or is freed outside it.

A replay repeats the launches of its capture on the same inputs, and results do not depend on timing, so every
comparison is exact.  Sizes are those that cut a sequence into several blocks' parts, which meet in the workspace."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def _inputs(dev, t, ctx, seed, hq=8, h=2, d=128, page=16):
    from blackwell_ops.decode import KVCacheInt8

    g = torch.Generator(device=dev).manual_seed(seed)
    cols = (ctx + t + page - 1) // page
    k, v = (torch.randint(-127, 128, (cols, h, page, d), generator=g, device=dev, dtype=torch.int8) for _ in "kv")
    ks, vs = ((torch.rand((cols, h, page), generator=g, device=dev) + 0.5) / 64 for _ in "kv")
    q = torch.randn((1, t, hq, d), generator=g, device=dev).half()
    table = torch.randperm(cols, generator=g, device=dev).to(torch.int32)[None]
    return q, KVCacheInt8(k, v, ks, vs), table, torch.tensor([ctx], dtype=torch.int32, device=dev)


def _fill(dev):
    """Takes the memory that is free, so that what a freed workspace held belongs to someone else."""
    return [torch.full((n,), 0x55, dtype=torch.uint8, device=dev) for n in (1 << 20, 3 << 20, 5 << 20, 12 << 20) for _ in range(4)]


def test_replay_after_the_workspace_has_grown(cuda_dev):
    from blackwell_ops.decode import tree_attention_int8

    small, big = _inputs(cuda_dev, 1, 5000, 1), _inputs(cuda_dev, 40, 3000, 2)
    want = tree_attention_int8(*small)
    st = torch.cuda.Stream(cuda_dev)
    st.wait_stream(torch.cuda.current_stream(cuda_dev))
    with torch.cuda.stream(st):
        tree_attention_int8(*small)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            out = tree_attention_int8(*small)
        large = tree_attention_int8(*big)
        others = _fill(cuda_dev)
        for _ in range(3):
            out.zero_()
            g.replay()
            st.synchronize()
            assert torch.equal(out, want)
    assert all(bool((x == 0x55).all()) for x in others)
    torch.cuda.synchronize(cuda_dev)
    assert torch.equal(large, tree_attention_int8(*big))


def test_second_graph_first(cuda_dev):
    """No warm-up, torch's own capture stream, the later graph replayed first, then both in turn."""
    from blackwell_ops.decode import tree_attention_int8

    a, b = _inputs(cuda_dev, 1, 4000, 3), _inputs(cuda_dev, 20, 2500, 4)
    junk = _fill(cuda_dev)
    del junk  # a fresh workspace does not come as zeros
    graphs, outs = [], []
    for args in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(tree_attention_int8(*args))
            outs.append(tree_attention_int8(*args))
        graphs.append(g)
    wa, wb = tree_attention_int8(*a), tree_attention_int8(*b)
    for x in (1, 0, 1, 1, 0):
        for o in outs:
            o.zero_()
        graphs[x].replay()
        torch.cuda.synchronize(cuda_dev)
        want = (wa, wb)[x]
        assert torch.equal(outs[2 * x], want) and torch.equal(outs[2 * x + 1], want)
        assert torch.equal(tree_attention_int8(*a), wa)


def test_two_graphs_on_two_streams(cuda_dev):
    """Captured one after the other on one stream, replayed side by side."""
    from blackwell_ops.decode import tree_attention_int8

    args = [_inputs(cuda_dev, 1, 6000 + 500 * i, 5 + i) for i in range(2)]
    want = [tree_attention_int8(*x) for x in args]
    graphs, outs = [], []
    for x in args:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append([tree_attention_int8(*x) for _ in range(20)])
        graphs.append(g)
    streams = [torch.cuda.Stream(cuda_dev) for _ in range(2)]
    torch.cuda.synchronize(cuda_dev)
    for _ in range(5):
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize(cuda_dev)
        for o, w in zip(outs, want):
            assert all(torch.equal(y, w) for y in o)


def test_growth_inside_a_capture(cuda_dev):
    """A small call, a larger one and the small one again in one graph, with other tensors between them."""
    from blackwell_ops.decode import tree_attention_int8

    small, big = _inputs(cuda_dev, 1, 5000, 8), _inputs(cuda_dev, 64, 2000, 9, hq=16)
    ws, wb = tree_attention_int8(*small), tree_attention_int8(*big)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a = tree_attention_int8(*small)
        b = tree_attention_int8(*big)
        x = torch.full((4 << 20,), 0x55, dtype=torch.uint8, device=cuda_dev)
        c = tree_attention_int8(*small)
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize(cuda_dev)
        assert torch.equal(a, ws) and torch.equal(b, wb) and torch.equal(c, ws) and bool((x == 0x55).all())
    from blackwell_ops import _lib

    assert _lib.device_status() == 0
