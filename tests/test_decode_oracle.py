"""CPU checks of the speculative-decoding operators' host side and oracle: frequencies against their formulas, the
fixed-point turns against 64-bit angles, the oracle's quantiser, tree masks and walk on cases worked by hand, and the C
entry points' refusals (made before any device call)."""
import math

import numpy as np
import pytest

from oracle import decode as ref

torch = pytest.importorskip("torch")


def test_frequencies():
    from blackwell_ops.decode import rotary_frequencies

    f, m = rotary_frequencies(8, 10000.0)
    assert m == 1.0 and np.allclose(f, [1, 0.1, 0.01, 0.001], rtol=1e-15)
    assert np.allclose(rotary_frequencies(8, 10000.0, {"type": "linear", "factor": 4.0})[0], f / 4, rtol=1e-15)
    # ntk: the lowest frequency is stretched by the factor, the highest kept
    n = rotary_frequencies(8, 10000.0, {"rope_type": "ntk", "factor": 4.0})[0]
    assert n[0] == 1 and np.isclose(n[-1], f[-1] / 4, rtol=1e-12)
    sc = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}
    g, f = rotary_frequencies(128, 500000.0, sc)[0].numpy(), rotary_frequencies(128, 500000.0)[0].numpy()
    wave = 2 * np.pi / f
    assert np.array_equal(g[wave < 8192 / 4], f[wave < 8192 / 4]) and np.allclose(g[wave > 8192], f[wave > 8192] / 8, rtol=1e-15)
    mid = (wave >= 8192 / 4) & (wave <= 8192)
    s = (8192 / wave[mid] - 1) / 3
    assert mid.any() and np.allclose(g[mid], (1 - s) * f[mid] / 8 + s * f[mid], rtol=1e-12)
    y, mag = rotary_frequencies(128, 10000.0, {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096})
    f = rotary_frequencies(128, 10000.0)[0]
    turns = 4096 * f / (2 * math.pi)
    assert mag == 0.1 * math.log(4.0) + 1
    assert torch.equal(y[turns > 40], f[turns > 40]) and torch.allclose(y[turns < 0.8], f[turns < 0.8] / 4, rtol=1e-15)
    assert rotary_frequencies(128, 1e4, {"rope_type": "yarn", "factor": 4.0, "attention_factor": 1.5,
                                         "original_max_position_embeddings": 4096})[1] == 1.5
    for bad in (lambda: rotary_frequencies(7), lambda: rotary_frequencies(0), lambda: rotary_frequencies(8, 0.5),
                lambda: rotary_frequencies(8, scaling={"rope_type": "x", "factor": 2}),
                lambda: rotary_frequencies(8, scaling={"rope_type": "llama3", "factor": 2})):
        with pytest.raises(RuntimeError):
            bad()


def test_fixed_point_turns():
    """pos * round(f / 2 pi * 2^64) modulo 2^64 is the angle's fraction of a turn to pos * 2^-54: the frequency's own
    64-bit rounding (53 bits) and no more."""
    from blackwell_ops.decode import rotary_frequencies

    for f in rotary_frequencies(128, 500000.0)[0].tolist():
        step = round(f / (2 * math.pi) * 2.0**64)
        for pos in (1, 4095, 131071, 2**31 - 1, -5):
            frac = (pos * step) % 2**64 / 2.0**64
            ang = math.fmod(pos * f / (2 * math.pi), 1.0) % 1.0
            assert min(abs(frac - ang), 1 - abs(frac - ang)) <= abs(pos) * 2.0**-52


def test_oracle_quantise_and_masks():
    q, s = ref.quantise(np.array([[127, 0.5, 1.5, -2.5, 126.5], [0, 0, 0, 0, 0], [np.nan, 1, -1, 0.5, 0], [np.inf, 1, 0, 0, 0]]))
    assert q[0].tolist() == [127, 0, 2, -2, 126] and s[0] == 1
    assert not q[1].any() and s[1] == 0
    assert q[2].tolist() == [0, 127, -127, 64, 0] and not q[3].any() and np.isinf(s[3])
    m, d = ref.tree_mask(np.array([[-1, 0, 0, 1, 3, -1, 6]]))
    assert m[0].tolist() == [1, 3, 5, 11, 27, 0, 0] and d[0].tolist() == [0, 1, 1, 2, 3, 0, 0]


def test_oracle_walk_by_hand():
    p = np.array([[[0.5, 0.3, 0.2, 0.0], [0.1, 0.9, 0, 0], [0.25] * 4]], dtype=np.float32)
    q = np.array([[[0.2, 0.8, 0, 0], [0.25] * 4, [0.25] * 4]], dtype=np.float32)
    one = np.ones((1, 4), dtype=np.float32)
    tok, star = np.array([[9, 1, 0]]), np.array([[-1, 0, 0]])
    # child 1: u q < p <=> 0.3 * 0.8 < 0.3: taken; its row's best follows
    n, path, out = ref.verify(p, tok, star, np.array([[0, 0.3, 0]], dtype=np.float32), one, q)
    assert n[0] == 1 and path[0].tolist() == [1, -1, -1] and out[0].tolist() == [1, 1, -1]
    # rejected at u = 0.5: w = [0.3, 0, 0.2, 0], Z = 0.5; child 2: 0.9 * 0.2 * 0.5 < 0.3: taken
    n, path, out = ref.verify(p, tok, star, np.array([[0, 0.5, 0.9]], dtype=np.float32), one, q)
    assert n[0] == 1 and path[0].tolist() == [2, -1, -1] and out[0].tolist() == [0, 0, -1]
    # drafts without a distribution: 0.5 < 0.3 no; Z = 0.7; 0.8 * 0.7 < 0.5 no; what is left is token 2
    n, path, out = ref.verify(p, tok, star, np.array([[0, 0.5, 0.8]], dtype=np.float32), one)
    assert n[0] == 0 and out[0].tolist() == [2, -1, -1]


def test_c_refusals():
    from blackwell_ops import _lib

    lib, bad = _lib.lib, _lib.BW_ERR_INVALID_ARGUMENT
    z3 = (0, 0, 0)
    rot = lambda dt=0, d=64, r=64, hq=1: lib.bw_rotary(None, *z3, hq, None, *z3, 0, None, None, dt, 1, 1, d, None, 0,  # noqa: E731
                                                       None, 1.0, r, 0, None)
    assert rot() == bad and b"null pointer" in lib.bw_last_error()
    assert rot(dt=2) == bad and b"fp16 or bf16" in lib.bw_last_error()
    assert rot(d=300) == bad and rot(r=63) == bad and rot(r=66) == bad and rot(hq=-1) == bad
    cache = (None,) * 4
    assert lib.bw_kv_read_int8(*cache, 1, 4, 2, 16, 300, None, 1, 1, None, None, 1, 1, None, None, 0, None) == bad
    assert lib.bw_kv_read_int8(*cache, 1, 4, 2, 16, 64, None, 1, 1, None, None, 1, 1, None, None, 0, None) == bad
    assert b"null" in lib.bw_last_error()
    assert lib.bw_kv_read_int8(*cache, 1, 0, 2, 16, 64, None, 0, 0, None, None, 0, 1, None, None, 0, None) == 0
    assert lib.bw_kv_move_int8(*cache, 1, 0, 2, 16, 64, None, 0, 0, None, None, 65, None, 0, 65, None) == bad
    assert lib.bw_tree_positions(None, 65, None, 1, 65, None, None, None) == bad
    assert lib.bw_tree_positions(None, 4, None, 0, 4, None, None, None) == 0
    att = lambda hq=4, dt=0, t=1: lib.bw_tree_attention_int8(None, *z3, dt, None, *cache, 0, 2, 16, 64, None, 0, 0,  # noqa: E731
                                                             None, None, None, 1, t, hq, 1.0, None, 0, None)
    assert att() == bad and b"null" in lib.bw_last_error()
    assert att(hq=3) == bad and att(dt=2) == bad and att(t=65) == bad
    assert lib.bw_verify_tree(None, None, None, None, None, None, 1, 1, 0, None, None, None, None) == bad
    assert lib.bw_verify_tree(None, None, None, None, None, None, 0, 1, 8, None, None, None, None) == 0


def test_lookup_tree():
    from blackwell_inference.spec_decode import lookup_tree

    # 1 2 3 4 | 1 2 3 5 | 1 2 3: continuations of (1 2 3), the later first
    tok, par = lookup_tree([1, 2, 3, 4, 1, 2, 3, 5, 1, 2, 3], 8, branches=2)
    assert tok[0] == 3 and par[0] == -1
    assert (tok[1], par[1]) == (5, 0) and 4 in tok and par[tok.index(4)] == 0
    assert all(0 <= p < i for i, p in enumerate(par) if i)
    assert lookup_tree([7], 8) == ([7], [-1]) and lookup_tree([1, 2, 1], 1) == ([1], [-1])
    tok, par = lookup_tree([9] * 40, 16)
    assert len(tok) <= 16 and set(tok) == {9}
