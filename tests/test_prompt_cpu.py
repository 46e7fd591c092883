"""Host side of the prompt's operators, and the arithmetic by which blocks of packed prompts are numbered: no GPU."""
import random

import pytest

torch = pytest.importorskip("torch")


def _edges(offsets, n):
    return [0, *(min(max(x, 0), n) for x in offsets), n]


def _block(offsets, n, p, slot):
    """Rows of block `slot`, found as a warp finds them (prompt_attention.cu: prompt_block); None: no rows."""
    edge = _edges(offsets, n)
    lo, hi = 0, len(offsets) + 1
    while hi - lo > 1:
        step = (hi - lo + 31) // 32
        before = [lo + lane * step < hi and edge[lo + lane * step] // p + lo + lane * step <= slot for lane in range(32)]
        last = max(lane for lane in range(32) if before[lane] or lane == 0)
        lo, hi = lo + last * step, min(hi, lo + (last + 1) * step)
    e0, e1 = edge[lo], edge[lo + 1]
    blocks = -(-(e1 - e0) // p) if e1 > e0 else 0
    i = slot - (e0 // p + lo)
    if i >= blocks:
        return None
    row0 = e0 + (blocks - 1 - i) * p
    return row0, min(row0 + p, e1), 1 <= lo < len(offsets)


def test_blocks_cover_every_row_once():
    """Each row lies in one block, blocks of real sequences do not leave theirs, and n / p + b + 2 numbers are enough."""
    rng = random.Random(1)
    for trial in range(400):
        p = rng.choice([1, 7, 16, 18, 36, 64, 128, 256])
        b = rng.choice([0, 1, 2, 5, 30, 31, 32, 33, 70, 200])
        lens = [rng.choice([0, 0, 1, 2, p - 1, p, p + 1, rng.randint(0, 5 * p)]) for _ in range(b)]
        first, spare = rng.choice([0, 0, 3, p, 2 * p + 1]), rng.choice([0, 0, 5, p, 3 * p - 1])
        offsets = [first]
        for m in lens:
            offsets.append(offsets[-1] + m)
        n = offsets[-1] + spare
        seen = [0] * n
        for slot in range(n // p + b + 2):
            got = _block(offsets, n, p, slot)
            if got is None:
                continue
            row0, row1, real = got
            assert row0 < row1 <= row0 + p
            owner = [i for i in range(b) if offsets[i] <= row0 < offsets[i + 1]]
            assert real == bool(owner)
            if real:
                assert row1 <= offsets[owner[0] + 1] and (row0 - offsets[owner[0]]) % p == 0
            for r in range(row0, row1):
                seen[r] += 1
        assert seen == [1] * n, (p, lens, first, spare)


def test_blocks_of_bad_offsets_stay_inside():
    rng = random.Random(2)
    for trial in range(300):
        n, b, p = rng.randint(1, 400), rng.randint(0, 80), rng.choice([7, 64, 128])
        offsets = [rng.randint(-50, 2 * n) for _ in range(b + 1)]
        for slot in range(n // p + b + 2):
            got = _block(offsets, n, p, slot)
            assert got is None or (0 <= got[0] < got[1] <= n and got[1] - got[0] <= p)


def test_arguments_before_any_device_call():
    from blackwell_ops import _lib

    lib, bad = _lib.lib, _lib.BW_ERR_INVALID_ARGUMENT

    def attention(dtype=0, b=1, n=4, hq=4, hk=2, d=64, st=256, scale=1.0):
        return lib.bw_prompt_attention(None, st, d, None, st, d, None, st, d, dtype, None, None, b, n, hq, hk, d, scale, None)

    for kw, word in (({"dtype": 2}, b"fp16 or bf16"), ({"b": -1}, b"b, n"), ({"n": -1}, b"b, n"), ({"hq": 3}, b"multiple"),
                     ({"hk": 0}, b"multiple"), ({"d": 257}, b"d <= 256"), ({"d": 0}, b"d <= 256"), ({"st": -1}, b"stride"),
                     ({}, b"null pointer"), ({"b": 2**40}, b"b, n"), ({"n": 2**40}, b"b, n")):
        assert attention(**kw) == bad and word in lib.bw_last_error(), kw
    assert attention(n=0) == 0

    def logprobs(dtype=0, ld=10, rows=3, v=10, top=2):
        return lib.bw_token_logprobs(None, dtype, ld, None, rows, v, top, None, None, None, None, None)

    for kw, word in (({"dtype": 3}, b"fp32"), ({"rows": -1}, b"rows"), ({"v": 0}, b"v <"), ({"v": 2**31}, b"v <"), ({"top": 33}, b"top"),
                     ({"top": 11}, b"top"), ({"top": -1}, b"top"), ({"ld": -1}, b"stride"), ({}, b"null pointer")):
        assert logprobs(**kw) == bad and word in lib.bw_last_error(), kw
    assert logprobs(rows=0) == 0

    def norm(dtype=0, b=1, t=3, d=64, eps=1e-6, rot=64, hq=2):
        return lib.bw_norm_rotary(None, 0, 128, 64, hq, None, 0, 0, 0, 0, None, None, dtype, b, t, d, None, None, eps, None, 0, None,
                                  1.0, rot, 0, None)

    for kw, word in (({"dtype": 2}, b"fp16 or bf16"), ({"d": 300}, b"d <="), ({"rot": 3}, b"even rot"), ({"rot": 66}, b"even rot"),
                     ({"hq": -1}, b"heads"), ({}, b"null pointer"), ({"hq": 0, "eps": -1.0, "rot": 0}, b"eps"),
                     ({"hq": 0, "eps": float("nan"), "rot": 0}, b"eps")):
        assert norm(**kw) == bad and word in lib.bw_last_error(), kw
    assert norm(b=0) == 0 and norm(t=0) == 0

    def write(b=1, t=3, counts=None, offsets=None, eps=1e-6, page=16, cols=1):
        return lib.bw_norm_rotary_kv_write_int8(None, 0, 0, 0, 0, None, 0, 0, 0, None, 0, 0, 0, None, None, 0, b, t, None, None, eps,
                                                None, 0, None, 1.0, 0, 0, None, None, None, None, 0, 2, page, 64, None, cols, cols,
                                                None, counts, offsets, None)

    for kw, word in (({"b": -1}, b"b < 2^31"), ({"b": 2**40}, b"b < 2^31"), ({"page": 0}, b"page >= 1"), ({}, b"null table"),
                     ({"cols": 0}, b"null pointer")):
        assert write(**kw) == bad and word in lib.bw_last_error(), kw
    assert write(t=0, cols=0) == 0 and write(b=0) == 0


def test_messages_on_the_host():
    from blackwell_ops import prompt as P

    x = torch.zeros((3, 2, 64), dtype=torch.float16)
    with pytest.raises(RuntimeError, match="q must be CUDA"):
        P.prompt_attention(x, x, x, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="logits must be CUDA"):
        P.token_logprobs(x[0], torch.zeros(2, dtype=torch.int64))


def test_prompts_of_the_decoder():
    """What packing refuses: tokens outside the vocabulary (which would fault in the embedding), long and nested prompts."""
    from types import SimpleNamespace

    from blackwell_inference.spec_decode import TreeSpeculativeDecoder

    dec = TreeSpeculativeDecoder.__new__(TreeSpeculativeDecoder)
    dec.dev, dec.max_len = torch.device("cpu"), 4
    dec.model = SimpleNamespace(base=SimpleNamespace(model=SimpleNamespace(embed_tokens=torch.nn.Embedding(10, 2))))
    tokens, lens = dec._pack([[0, 9], [], torch.tensor([3], dtype=torch.int32)])
    assert tokens.tolist() == [0, 9, 3] and lens == [2, 0, 1]
    assert dec._pack([])[0].numel() == 0 and dec._pack([[]])[1] == [0]
    for match, prompts in [("0 to 9", [[1], [10]]), ("0 to 9", [[-1, 2]]), ("max_len = 4", [[1] * 5]), ("list of tokens", [[[1]]])]:
        with pytest.raises(RuntimeError, match=match):
            dec._pack(prompts)
