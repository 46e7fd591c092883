"""The prompt operators as programs call them: on two streams at once, in captured graphs that take turns, on outputs and
inputs that lie inside other memory.  Results are compared with those of the same call alone, bit for bit: none of the
kernels adds in an order that varies."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def _randn(seed, shape, dt, dev):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dt).to(dev)


def _off(lens, dev):
    return torch.tensor([0, *lens]).cumsum(0).to(torch.int32).to(dev)


def _calls(dev):
    """Calls of each operator whose kernels differ, as functions without arguments that return lists of tensors."""
    from blackwell_ops.decode import KVCacheInt8, norm_rotary, norm_rotary_kv_write_int8, rotary_plan
    from blackwell_ops.prompt import prompt_attention, token_logprobs

    lens = [700, 1, 0, 333, 513]
    n, off = sum(lens), _off(lens, dev)
    calls = []
    for hq, hk, d, dt in ((16, 8, 128, torch.bfloat16), (28, 4, 64, torch.float16), (4, 2, 80, torch.float16)):
        q, k, v = (_randn(s, (n, h, d), dt, dev) for s, h in ((1, hq), (2, hk), (3, hk)))
        calls.append(lambda q=q, k=k, v=v: [prompt_attention(q, k, v, off)])
    for rows, v, dt, top in ((3, 50257, torch.bfloat16, 20), (100, 3001, torch.float32, 5), (600, 4097, torch.float16, 1)):
        x, tok = _randn(4, (rows, v), dt, dev), torch.arange(rows, device=dev)
        calls.append(lambda x=x, tok=tok, top=top: list(token_logprobs(x, tok, top)))
    q, k, v = (_randn(s, (n, h, 128), torch.float16, dev) for s, h in ((5, 16), (6, 8), (7, 8)))
    w, pos = _randn(8, (128,), torch.float16, dev), torch.arange(n, dtype=torch.int32, device=dev)
    plan = rotary_plan(128, device=dev)
    calls.append(lambda: list(norm_rotary(q, k, pos, plan, w, w)))
    pages = 5 * 11
    table = torch.arange(pages, dtype=torch.int32, device=dev).view(5, 11)
    start = torch.zeros(5, dtype=torch.int32, device=dev)

    def write():
        cache = KVCacheInt8(*(torch.zeros((pages, 8, 64, 128), dtype=torch.int8, device=dev) for _ in range(2)),
                            *(torch.zeros((pages, 8, 64), device=dev) for _ in range(2)))
        out = norm_rotary_kv_write_int8(q, k, v, pos, plan, cache, table, start, w, w, offsets=off, keys=True)
        return [*out, cache.k, cache.v, cache.k_scale, cache.v_scale]

    calls.append(write)
    return calls


def test_two_streams_at_once(cuda_dev):
    """Every operator beside every other one, and beside itself."""
    calls = _calls(cuda_dev)
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(cuda_dev) for _ in range(2)]
    got = []
    for i in range(len(calls)):
        for j in range(i, len(calls)):
            for st, c in zip(streams, (i, j)):
                with torch.cuda.stream(st):
                    got += [(c, calls[c]()) for _ in range(2)]
    torch.cuda.synchronize()
    for c, y in got:
        assert all(torch.equal(a, b) for a, b in zip(y, want[c])), c


def test_graphs_that_take_turns(cuda_dev):
    """Two graphs of all operators, replayed one after the other and at once, next to calls without a graph."""
    calls = _calls(cuda_dev)
    want = [c() for c in calls]
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = [c() for c in calls]
        graphs.append((g, out))
    streams = [torch.cuda.Stream(cuda_dev) for _ in range(2)]
    torch.cuda.synchronize()
    for at_once in (False, True):
        for _, out in graphs:
            for y in out:
                for x in y:
                    x.zero_()
        torch.cuda.synchronize()
        for st, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
                g.replay()
            if not at_once:
                st.synchronize()
        eager = [c() for c in calls]
        torch.cuda.synchronize()
        for y in [graphs[0][1], graphs[1][1], eager]:
            assert all(torch.equal(a, b) for got, w in zip(y, want) for a, b in zip(got, w))


@pytest.mark.parametrize("hq,hk,d", [(16, 8, 128), (28, 4, 64), (4, 2, 80)])
def test_memory_around(cuda_dev, hq, hk, d):
    """Rows before and behind the packed ones are neither read (NaN there changes nothing) nor written, whatever the
    offsets hold."""
    from blackwell_ops._lib import DTYPE_CODE, lib
    from blackwell_ops.prompt import prompt_attention

    n, edge, dt = 300, 300, torch.float16
    q, k, v = (_randn(s, (n, h, d), dt, cuda_dev) for s, h in ((1, hq), (2, hk), (3, hk)))
    inside = []
    for x in (q, k, v):
        y = torch.full((n + 2 * edge, *x.shape[1:]), float("nan"), dtype=dt, device=cuda_dev)
        y[edge:-edge] = x
        inside.append(y[edge:-edge])
    out = torch.empty((n + 2 * edge, hq, d), dtype=dt, device=cuda_dev)
    for off in ([0, 300], [0, 129, 130, 300], [7, 140, 290], [0, 200, 100, 300], [5, 500, 1000, 2000], [-7, 3, -100, 12],
                [300, 0, 300, 0], [-5, 305]):
        offsets = torch.tensor(off, dtype=torch.int32, device=cuda_dev)
        out.fill_(7.0)
        args = [a for x in inside for a in (x.data_ptr(), x.stride(0), x.stride(1))]
        status = lib.bw_prompt_attention(*args, DTYPE_CODE[dt], out[edge:].data_ptr(), offsets.data_ptr(), len(off) - 1, n, hq, hk,
                                         d, d ** -0.5, torch.cuda.current_stream(cuda_dev).cuda_stream)
        assert status == 0
        assert bool((out[:edge] == 7).all()) and bool((out[-edge:] == 7).all())
        if off == sorted(off):
            assert torch.equal(out[edge:-edge], prompt_attention(q, k, v, offsets)) and bool(torch.isfinite(out).all())


@pytest.mark.parametrize("dt", [torch.float16, torch.float32])
def test_logits_around(cuda_dev, dt):
    """Rows of a wider matrix whose other columns are NaN, from every start within 32 bytes; rows that are the same row."""
    from blackwell_ops.prompt import token_logprobs

    x = _randn(1, (7, 1003), dt, cuda_dev)
    tok = torch.arange(7, device=cuda_dev) * 100
    want = token_logprobs(x, tok, 6)
    for at in range(17):
        wide = torch.full((7, 1003 + 37), float("nan"), dtype=dt, device=cuda_dev)
        wide[:, at:at + 1003] = x
        got = token_logprobs(wide[:, at:at + 1003], tok, 6)
        # Another start puts other logits into a thread.  Either sum has at most 20 roundings of 2^-24 and exponentials off by
        # 2^-20 (their arguments, at most 12, rounded): 2^-18 of S apart, and as much of the values that are formed from ln S.
        assert torch.equal(got.top_tokens, want.top_tokens)
        for a, b in ((got.logprobs, want.logprobs), (got.entropy, want.entropy), (got.top_logprobs, want.top_logprobs)):
            assert bool(((a - b).abs() <= 2.0**-20 * (1 + b.abs()) * 4).all())
    one = token_logprobs(x[3:4].expand(7, -1), tok, 6)
    assert all(bool((y == y[:1]).all()) for y in (one.entropy, one.top_logprobs, one.top_tokens))
    assert torch.equal(one.top_logprobs[0], want.top_logprobs[3])


def test_the_decoder_keeps_its_lengths_in_place(cuda_dev):
    transformers = pytest.importorskip("transformers")
    from blackwell_inference.spec_decode import TreeSpeculativeDecoder
    from test_gpu_spec_decode_configs import SMALL, _pair

    mdl, _ = _pair(transformers.Qwen3Config(**SMALL), cuda_dev)
    dec = TreeSpeculativeDecoder(mdl, batch=2, max_len=50, packed=True)
    ctx = dec.ctx
    dec.prefill_packed([[1, 2, 3], [4]])
    assert dec.ctx is ctx and ctx.tolist() == [3, 1]
    with pytest.raises(RuntimeError, match="tokens must be"):
        dec.prefill_packed([[1, 512], [4]])
    assert ctx.tolist() == [3, 1]  # a refused call changes nothing
