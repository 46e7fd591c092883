"""Cases of the speculative-decoding operators: rotary positions, the paged int8 KV cache, attention of a tree of
drafted tokens over that cache, and the verification of the drafted tokens.

Sizes are those of the decoders this repository already names (Qwen3-0.6B: 16 query / 8 key heads, vocabulary 151936;
Llama-3-8B: 32 / 8; Llama-3-70B: 64 / 8; head dimension 128) and generic ones; the cache's pages are scattered as a
server's allocator leaves them, and the sequences of a batch have different lengths.

Conventions shared by every case: the cache is four tensors, int8 codes k, v [.., pages, heads, page, D] and one fp32
scale per token and head [.., pages, heads, page]; slot s of sequence b is row s % page of page table[b, s // page].
"""
import math
import sys

import torch

own = False

DT = {"f16": torch.float16, "bf16": torch.bfloat16}
LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}
YARN = {"rope_type": "yarn", "factor": 4.0, "beta_fast": 32.0, "beta_slow": 1.0,
        "original_max_position_embeddings": 32768}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step's rotation of a small batch: pure latency
        dict(name="rotary decode 16", op="rotary", tokens=16, hq=16, hk=8, d=128, rot=128, layout="half",
             scaling="none", maxpos=4096, dt="f16"),
        # a chunk of a long prompt, 70B heads, frequencies scaled for long contexts
        dict(name="rotary prefill 8191", op="rotary", tokens=8191, hq=64, hk=8, d=128, rot=128, layout="half",
             scaling="llama3", maxpos=131072, dt="bf16"),
        # one decode step's new keys and values of 64 sequences, quantised into the cache and read back
        dict(name="cache write decode 64", op="write", b=64, t=1, hq=0, hk=8, d=128, page=16, ctx=4001, rot=0,
             layout="half", scaling="none", dt="f16"),
        # a prefill chunk of two sequences: rotation fused with the write, read back for the chunk's own attention
        dict(name="cache rotary write chunk", op="write", b=2, t=2048, hq=32, hk=8, d=128, page=64, ctx=6144, rot=128,
             layout="half", scaling="llama3", dt="bf16"),
        # four long contexts read back as 16-bit values (handing a cache over to a dense attention)
        dict(name="cache read 4 x 16k", op="read", b=4, hk=8, d=128, page=16, ctx=16383, dt="bf16"),
        # accepted draft nodes moved to their final slots in all 28 layers, then read back
        dict(name="cache move 28 layers", op="move", layers=28, b=32, t=16, hk=8, d=128, page=16, ctx=1021, dt="f16"),
        # one new token of one short sequence: latency
        dict(name="attention 1 token 1k", op="attention", b=1, t=1, hq=16, hk=8, d=128, page=16, ctx=1023,
             tree="chain", dt="f16"),
        # ordinary batched decode, ragged lengths: bound by the cache's bytes
        dict(name="attention decode 64 x 4k", op="attention", b=64, t=1, hq=32, hk=8, d=128, page=16, ctx=4095,
             tree="chain", dt="bf16"),
        # a tree of 24 drafted tokens in each of eight sequences, head dimension 64
        dict(name="attention tree 24, 8 x 8k", op="attention", b=8, t=24, hq=32, hk=8, d=64, page=64, ctx=8190,
             tree="random", dt="f16"),
        # a full tree of 64 nodes over one very long context, 70B heads: bound by arithmetic
        dict(name="attention tree 64, 128k", op="attention", b=1, t=64, hq=64, hk=8, d=128, page=64, ctx=131008,
             tree="random", dt="bf16"),
        # one sequence's chain of four drafts from a draft model
        dict(name="verify chain 5", op="verify", b=1, t=5, v=151936, tree="chain", drafts=True),
        # a batch of trees whose drafts were looked up (no draft distribution)
        dict(name="verify tree 16 x 32", op="verify", b=32, t=16, v=151936, tree="binary", drafts=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw(rng):
    op = rng.choice(["rotary", "write", "read", "move", "attention", "attention", "attention", "verify"])
    dt = rng.choice(["f16", "bf16"])
    hq, hk = rng.choice([(16, 8), (32, 8), (64, 8), (8, 8), (28, 4), (12, 1)])
    d = rng.choice([64, 128])
    page = rng.choice([16, 32, 64, 128])
    layout, scaling = rng.choice(["half", "interleaved"]), rng.choice(["none", "llama3", "yarn"])
    rot = rng.choice([d, d, d // 2])
    if op == "rotary":
        return dict(op=op, tokens=_log(rng, 1, 8191), hq=hq, hk=hk, d=d, rot=rot, layout=layout, scaling=scaling,
                    maxpos=_log(rng, 1024, 131072), dt=dt)
    if op == "write":
        b = _log(rng, 1, 64)
        fused = rng.random() < 0.5
        return dict(op=op, b=b, t=_log(rng, 1, max(1, 4096 // b)), hq=hq if fused else 0, hk=hk, d=d, page=page,
                    ctx=_log(rng, 1, 8192), rot=rot if fused else 0, layout=layout,
                    scaling=scaling if fused else "none", dt=dt)
    if op == "read":
        return dict(op=op, b=_log(rng, 1, 64), hk=hk, d=d, page=page, ctx=_log(rng, 1, 16384), dt=dt)
    if op == "move":
        return dict(op=op, layers=rng.choice([1, 16, 28, 32]), b=_log(rng, 1, 64), t=rng.randint(3, 64), hk=hk, d=d,
                    page=page, ctx=_log(rng, 1, 2048), dt=dt)
    if op == "attention":
        return dict(op=op, b=_log(rng, 1, 64), t=rng.choice([1, 1, _log(rng, 2, 64)]), hq=hq, hk=hk, d=d, page=page,
                    ctx=_log(rng, 1, 131008), tree=rng.choice(["chain", "binary", "random"]), dt=dt)
    return dict(op=op, b=_log(rng, 1, 64), t=rng.randint(1, 24), v=rng.choice([32000, 50257, 128256, 151936]),
                tree=rng.choice(["chain", "binary", "random"]), drafts=rng.random() < 0.5)


# a state holds its cache (or probabilities), so a drawn one is bounded in size as well as in work
MOST = {"rotary": 302e6, "write": 109e6, "read": 331e6, "move": 109e6, "attention": 4.19e8, "verify": 3.12e8}


def draw(rng):
    while True:
        c = _draw(rng)
        w = work(c)
        if c["op"] == "verify":
            size = c["b"] * c["t"] * c["v"] * 4 * (2 if c["drafts"] else 1)
        elif c["op"] == "move":
            size = 2 * c["layers"] * c["b"] * (c["ctx"] + c["t"]) * c["hk"] * c["d"]
            size = max(w["bytes"], size / 16)  # the cache it lies in
        else:
            size = w["bytes"]
        if size <= MOST[c["op"]] and w["flops"] <= 2.8e11:
            return c


def _lens(c):
    """Context lengths of a batch: from half of ctx to all of it, the same for every seed."""
    return [max(1, c["ctx"] - (c["ctx"] // 2) * i // c["b"]) for i in range(c["b"])]


def _taken(c):
    """Accepted nodes of each sequence of a move: none to all that fit, nodes whose slots are not targets."""
    most = (c["t"] - 1) // 2
    return [i % (most + 1) for i in range(1, c["b"] + 1)]


def work(c):
    op = c["op"]
    if op == "rotary":
        n = c["tokens"] * (c["hq"] + c["hk"]) * c["d"]
        return {"bytes": 4 * n + 4 * c["tokens"], "flops": 3 * n}
    if op == "write":  # 16-bit in, codes and scales written, 16-bit values read back
        rows = c["b"] * c["t"] * c["hk"] * 2
        q = c["b"] * c["t"] * c["hq"] * c["d"]
        return {"bytes": rows * (c["d"] * 5 + 4) + 4 * q, "flops": 4 * rows * c["d"] + 3 * q}
    if op == "read":
        rows = sum(_lens(c)) * c["hk"] * 2
        return {"bytes": rows * (3 * c["d"] + 4), "flops": rows * c["d"]}
    if op == "move":
        rows = c["layers"] * c["hk"] * 2
        moved, back = sum(_taken(c)), c["b"] * c["t"]
        return {"bytes": rows * (moved * 2 * (c["d"] + 4) + back * 2 * c["d"]), "flops": rows * moved * c["d"]}
    if op == "attention":
        keys = sum(_lens(c)) + c["b"] * c["t"]
        qo = 4 * c["b"] * c["t"] * c["hq"] * c["d"]
        return {"bytes": keys * c["hk"] * (2 * c["d"] + 8) + qo, "flops": 4 * c["t"] * c["hq"] * c["d"] * keys}
    rows = 3 if c["drafts"] else 2  # target, draft, noise: the row at which the walk ends
    return {"bytes": c["b"] * c["v"] * 4 * rows + 40 * c["b"] * c["t"], "flops": 3 * c["b"] * c["v"]}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)


def _normal(g, shape, dt):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dt)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _table(g, b, slots, page):
    """Scattered pages: every sequence's pages anywhere in the cache."""
    per = -(-slots // page)
    pages = b * per + 3
    return torch.randperm(pages, generator=g, device="cuda")[: b * per].to(torch.int32).view(b, per), pages


def _cache(g, lead, pages, c):
    shape = (*lead, pages, c["hk"], c["page"], c["d"])
    kv = []
    for _ in range(2):
        x = torch.empty(shape, dtype=torch.float16, device="cuda").normal_(generator=g)
        kv.append(x.mul_(32).round_().clamp_(-127, 127).to(torch.int8))
    sc = [(torch.rand(shape[:-1], generator=g, device="cuda") + 0.5) / 32 for _ in range(2)]
    return kv[0], kv[1], sc[0], sc[1]


def _handle(s):
    """The framework's handle of the cache, which a program keeps as long as the cache."""
    if own:
        s["kv"] = _ops().KVCacheInt8(*s["cache"])


def _parents(g, b, t, tree):
    if tree == "chain":
        p = torch.arange(t, device="cuda") - 1
        return p.to(torch.int32).expand(b, t).contiguous()
    i = torch.arange(t, device="cuda")
    if tree == "binary":
        p = (i - 1).div(2, rounding_mode="floor")
    else:  # most drafts hang from recent nodes
        u = torch.rand((b, t), generator=g, device="cuda")
        p = (i - 1 - (u * u * i.clamp(max=6)).long()).clamp(min=0)
    p = torch.where(i == 0, -1, p)
    return p.to(torch.int32).expand(b, t).contiguous()


def _ancestors(parents):
    """Bit j of [b, i]: node j is node i or one of its ancestors (an int64 holds 64 nodes)."""
    t = parents.shape[1]
    up = parents.long()
    bits = (torch.ones_like(up) << torch.arange(t, device="cuda")).contiguous()
    for _ in range(6):
        ok = up >= 0
        at = up.clamp(min=0)
        bits = bits | torch.where(ok, bits.gather(1, at), 0)
        up = torch.where(ok, up.gather(1, at), -1)
    return bits


def _scaling(c):
    return {"none": None, "llama3": LLAMA3, "yarn": YARN}[c["scaling"]]


def _frequencies(c):
    """Radians per position of each rotated pair, and the magnitude of the rotated pair (64-bit floats)."""
    base, half, sc = 500000.0, c["rot"] // 2, _scaling(c)
    f = base ** (-torch.arange(half, dtype=torch.float64) * 2.0 / c["rot"])
    if sc is None:
        return f, 1.0
    old, factor = sc["original_max_position_embeddings"], sc["factor"]
    if sc["rope_type"] == "llama3":
        lo, hi = sc["low_freq_factor"], sc["high_freq_factor"]
        mix = ((old * f / (2 * math.pi) - lo) / (hi - lo)).clamp(0, 1)
        return f * ((1 - mix) / factor + mix), 1.0
    dim = lambda turns: c["rot"] * math.log(old / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    lo, hi = max(math.floor(dim(sc["beta_fast"])), 0), min(math.ceil(dim(sc["beta_slow"])), c["rot"] - 1)
    ramp = ((torch.arange(half, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
    return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0


def _plan(s, c):
    """The rotation's frequencies as a program holds them: a table for the plain form, the framework's plan."""
    f, m = _frequencies(c)
    s["freq"], s["mag"] = f.float().cuda(), m
    if own:
        s["plan"] = _ops().rotary_plan(c["rot"], base=500000.0, scaling=_scaling(c),
                                       interleaved=c["layout"] == "interleaved", device="cuda")


def _ops():
    if "blackwell-inference-server_b200" not in sys.path:
        sys.path.insert(1, "blackwell-inference-server_b200")
    import blackwell_ops.decode as ops
    return ops


def prepare(c, seed):
    g, op = _gen(seed), c["op"]
    s = {"c": c}
    if op == "rotary":
        _plan(s, c)
        s["q"] = _normal(g, (c["tokens"], c["hq"], c["d"]), DT[c["dt"]])
        s["k"] = _normal(g, (c["tokens"], c["hk"], c["d"]), DT[c["dt"]])
        s["pos"] = torch.randint(0, c["maxpos"], (c["tokens"],), generator=g, device="cuda", dtype=torch.int32)
    elif op == "write":
        if c["rot"]:
            _plan(s, c)
        s["table"], pages = _table(g, c["b"], c["ctx"] + c["t"], c["page"])
        s["cache"], s["start"] = _cache(g, (), pages, c), _i32(_lens(c))
        # queries, keys and values lie side by side, as one projection leaves them
        h = c["hq"] + 2 * c["hk"]
        s["qkv"] = _normal(g, (c["b"], c["t"], h, c["d"]), DT[c["dt"]])
        s["pos"] = s["start"][:, None] + torch.arange(c["t"], device="cuda", dtype=torch.int32)
    elif op == "read":
        s["table"], pages = _table(g, c["b"], c["ctx"], c["page"])
        s["cache"], s["lens"] = _cache(g, (), pages, c), _i32(_lens(c))
    elif op == "move":
        s["table"], pages = _table(g, c["b"], c["ctx"] + c["t"], c["page"])
        s["cache"], s["start"] = _cache(g, (c["layers"],), pages, c), _i32(_lens(c))
        n = _taken(c)
        s["n"] = _i32(n)
        # accepted nodes in ascending order, all beyond the slots they move to
        r = torch.rand((c["b"], c["t"]), generator=g, device="cuda")
        i = torch.arange(c["t"], device="cuda")
        r = torch.where(i <= s["n"][:, None], 2.0, r).argsort(1)
        path = torch.where(i < s["n"][:, None], r, c["t"]).sort(1).values
        s["path"] = torch.where(path < c["t"], path, -1).to(torch.int32)
    elif op == "attention":
        s["table"], pages = _table(g, c["b"], c["ctx"] + c["t"], c["page"])
        s["cache"], s["lens"] = _cache(g, (), pages, c), _i32(_lens(c))
        s["q"] = (2.5 * _normal(g, (c["b"], c["t"], c["hq"], c["d"]), torch.float32)).to(DT[c["dt"]])
        s["mask"] = _ancestors(_parents(g, c["b"], c["t"], c["tree"]))
    else:
        b, t, v = c["b"], c["t"], c["v"]
        z = torch.empty((b, t, v), device="cuda").normal_(generator=g).mul_(3.0)
        s["p"] = z.softmax(-1)
        qz = z.add_(torch.empty_like(z).normal_(generator=g), alpha=0.7).softmax(-1)
        s["parents"] = _parents(g, b, t, c["tree"])
        up = s["parents"].long().clamp(min=0)
        # each drafted token is a draw from the draft model's distribution at its parent
        tok = [(qz[i, up[i]] / torch.empty((t, v), device="cuda").exponential_(generator=g)).argmax(-1)
               for i in range(b)]
        s["tokens"] = torch.stack(tok)
        s["q"] = qz if c["drafts"] else None
        s["u"] = torch.rand((b, t), generator=g, device="cuda")
        s["e"] = torch.empty((b, v), device="cuda").exponential_(generator=g)
    if "cache" in s:
        _handle(s)
    return s


# ------------------------------------------------------------------ the framework's calls and the plain forms
def run(s):
    return (_own if own else _plain)(s, s["c"])


def _own(s, c):
    ops = _ops()
    op = c["op"]
    if op == "rotary":
        return ops.rotary(s["q"], s["k"], s["pos"], s["plan"])
    if op == "write":
        q, k, v = s["qkv"].split([c["hq"], c["hk"], c["hk"]], dim=2)
        out = {}
        if c["rot"]:
            out["q"] = ops.rotary_kv_write_int8(q, k, v, s["pos"], s["plan"], s["kv"], s["table"], s["start"])
        else:
            ops.kv_write_int8(k, v, s["kv"], s["table"], s["start"])
        out["k"], out["v"] = ops.kv_read_int8(s["kv"], s["table"], s["start"], c["t"], dtype=DT[c["dt"]])
        out["ks"], out["vs"] = s["cache"][2:]
        return out
    if op == "read":
        return ops.kv_read_int8(s["kv"], s["table"], None, c["ctx"], lens=s["lens"], dtype=DT[c["dt"]])
    if op == "move":
        ops.kv_move_int8(s["kv"], s["table"], s["start"], s["path"], s["n"])
        return ops.kv_read_int8(s["kv"], s["table"], s["start"], c["t"], dtype=DT[c["dt"]])
    if op == "attention":
        return ops.tree_attention_int8(s["q"], s["kv"], s["table"], s["lens"], s["mask"])
    return ops.verify_tree(s["p"], s["tokens"], s["parents"], s["u"], s["e"], draft_probs=s["q"])


def _turn(x, pos, s, c):
    """The rotation in 32 bits; x [.., heads, D], pos [..]."""
    x = x.float()
    a = pos.float()[..., None, None] * s["freq"]
    co, si = torch.cos(a) * s["mag"], torch.sin(a) * s["mag"]
    r = c["rot"]
    if c["layout"] == "half":
        x1, x2 = x[..., : r // 2], x[..., r // 2 : r]
        y = torch.cat([x1 * co - x2 * si, x1 * si + x2 * co], -1)
    else:
        x1, x2 = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack([x1 * co - x2 * si, x1 * si + x2 * co], -1).flatten(-2)
    return torch.cat([y, x[..., r:]], -1)


def _slots(s, c, start, count):
    """Page and row of slots start .. start + count of each sequence, [b, count]."""
    at = start.long()[:, None] + torch.arange(count, device="cuda")
    return s["table"].long().gather(1, at // c["page"]), at % c["page"]


def _plain_read(s, c, start, count, dt):
    page, row = _slots(s, c, start, count)
    out = []
    for codes, scale in ((s["cache"][0], s["cache"][2]), (s["cache"][1], s["cache"][3])):
        out.append((codes[page, :, row].float() * scale[page, :, row][..., None]).to(dt))
    return out


def _plain(s, c):
    op = c["op"]
    if op == "rotary":
        dt = DT[c["dt"]]
        return _turn(s["q"], s["pos"], s, c).to(dt), _turn(s["k"], s["pos"], s, c).to(dt)
    if op == "write":
        dt = DT[c["dt"]]
        q, k, v = s["qkv"].split([c["hq"], c["hk"], c["hk"]], dim=2)
        out = {}
        k, v = k.float(), v.float()
        if c["rot"]:
            out["q"] = _turn(q, s["pos"], s, c).to(dt)
            k = _turn(k, s["pos"], s, c)
        page, row = _slots(s, c, s["start"], c["t"])
        for x, codes, scale in ((k, s["cache"][0], s["cache"][2]), (v, s["cache"][1], s["cache"][3])):
            sc = x.abs().amax(-1) / 127
            codes[page, :, row, :] = torch.round(x / sc[..., None]).clamp(-127, 127).to(torch.int8)
            scale[page, :, row] = sc
        out["k"], out["v"] = _plain_read(s, c, s["start"], c["t"], dt)
        out["ks"], out["vs"] = s["cache"][2:]
        return out
    if op == "read":
        zero = torch.zeros_like(s["lens"])
        keep = (torch.arange(c["ctx"], device="cuda") < s["lens"][:, None])[..., None, None]
        return [torch.where(keep, x, 0) for x in _plain_read(s, c, zero, c["ctx"], DT[c["dt"]])]
    if op == "move":
        page, row = _slots(s, c, s["start"], c["t"])
        i = torch.arange(c["t"], device="cuda")
        # the row that ends up at slot start + i: an accepted node's, or the one that is there
        src = torch.where((i >= 1) & (i <= s["n"][:, None]), s["path"].long().roll(1, 1), i)
        fp, fr = page.gather(1, src), row.gather(1, src)
        for x in s["cache"]:
            for layer in x:
                layer[page, :, row] = layer[fp, :, fr]
        both = [_plain_read({**s, "cache": [x[i] for x in s["cache"]]}, c, s["start"], c["t"], DT[c["dt"]])
                for i in range(c["layers"])]
        return [torch.stack(x) for x in zip(*both)]
    if op == "attention":
        return _plain_attention(s, c)
    return _plain_verify(s, c)


def _plain_attention(s, c):
    b, t, hk, d = c["b"], c["t"], c["hk"], c["d"]
    grp, n = c["hq"] // hk, c["ctx"] + c["t"]
    k, v = _plain_read(s, c, torch.zeros_like(s["lens"]), n, torch.float32)
    q = s["q"].float().view(b, t, hk, grp, d).permute(0, 2, 3, 1, 4).reshape(b, hk, grp * t, d)
    score = (q @ k.permute(0, 2, 3, 1)).view(b, hk, grp, t, n) / math.sqrt(d)
    node = torch.arange(n, device="cuda") - s["lens"].long()[:, None]  # [b, n]: node index of a slot, < 0: context
    bit = (s["mask"][:, :, None] >> node.clamp(0, t - 1)[:, None, :]) & 1
    seen = (node[:, None, :] < 0) | ((node[:, None, :] < t) & (bit != 0))
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    w = torch.exp(score - top)
    w = w / w.sum(-1, keepdim=True).clamp(min=1e-30)
    o = w.view(b, hk, grp * t, n) @ v.permute(0, 2, 1, 3)
    return o.view(b, hk, grp, t, d).permute(0, 3, 1, 2, 4).reshape(b, t, c["hq"], d).to(DT[c["dt"]])


def _plain_verify(s, c):
    b, t, v = c["b"], c["t"], c["v"]
    p, q, tok, at = s["p"], s["q"], s["tokens"], torch.arange(b, device="cuda")
    cur = torch.zeros(b, dtype=torch.long, device="cuda")
    n = torch.zeros(b, dtype=torch.long, device="cuda")
    path = torch.full((b, t), -1, dtype=torch.long, device="cuda")
    w, z = p[:, 0], torch.ones(b, device="cuda")
    for i in range(1, t):  # nodes in order: the walk is at `cur`, and a node counts only if it hangs from there
        child = s["parents"][:, i] == cur
        x = tok[:, i]
        wx = w.gather(1, x[:, None])[:, 0]
        qrow = q[at, cur] if q is not None else None
        qx = qrow.gather(1, x[:, None])[:, 0] if q is not None else torch.ones_like(wx)
        take = child & (s["u"][:, i] * qx * z < wx)
        drop = child & ~take
        if q is not None:
            rest = (w - z[:, None] * qrow).clamp(min=0)
        else:
            rest = w.scatter(1, x[:, None], 0.0)
        z = torch.where(take, 1.0, torch.where(drop, rest.sum(-1), z))
        w = torch.where(take[:, None], p[:, i], torch.where(drop[:, None], rest, w))
        path = torch.where(take[:, None] & (torch.arange(t, device="cuda") == n[:, None]), i, path)
        n = n + take
        cur = torch.where(take, i, cur)
    w = torch.where((w > 0).any(-1, keepdim=True), w, p[at, cur])
    score = torch.where(w > 0, w / s["e"], -1.0)
    idx = torch.arange(v, device="cuda")
    last = torch.where(score == score.amax(-1, keepdim=True), idx, v).amin(-1)
    out = torch.where(path >= 0, tok.gather(1, path.clamp(min=0)), -1)
    out = torch.where(torch.arange(t, device="cuda") == n[:, None], last[:, None], out)
    return n.to(torch.int32), path.to(torch.int32), out


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_rotate(x, pos, c):
    f, m = _frequencies(c)
    ang = pos.double()[..., None, None] * f.cuda()
    unit = m * torch.polar(torch.ones_like(ang), ang)
    r, y = c["rot"], x.double().clone()
    first = slice(0, r // 2) if c["layout"] == "half" else slice(0, r, 2)
    second = slice(r // 2, r) if c["layout"] == "half" else slice(1, r, 2)
    z = torch.complex(x[..., first].double(), x[..., second].double()) * unit
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_rows(x, s, c, b, lo, hi):
    """Values of slots lo .. hi of sequence b in 64 bits, [hi - lo, heads, d]; x: a pair of codes and scales."""
    pages = s["table"][b].long()
    codes, scale = (y[pages].movedim(2, 1).flatten(0, 1) for y in x)  # [slots, heads, ..]
    return codes[lo:hi].double() * scale[lo:hi].double()[..., None]


def exact(c, seed):
    op = c["op"]
    if op == "verify":
        return None
    s = prepare(c, seed)
    if op == "rotary":
        return _exact_rotate(s["q"], s["pos"], c), _exact_rotate(s["k"], s["pos"], c)
    ck, cv, sk, sv = s["cache"]
    if op == "write":
        out = {}
        hq, hk = c["hq"], c["hk"]
        k, v = s["qkv"][:, :, hq : hq + hk].double(), s["qkv"][:, :, hq + hk :].double()
        if c["rot"]:
            out["q"] = _exact_rotate(s["qkv"][:, :, :hq], s["pos"], c)
            k = _exact_rotate(s["qkv"][:, :, hq : hq + hk], s["pos"], c)
        for name, x, scale in (("k", k, sk.double()), ("v", v, sv.double())):
            step = x.abs().max(-1).values / 127
            out[name] = torch.round(x / step[..., None]) * step[..., None]
            for i, first in enumerate(_lens(c)):
                slot = torch.arange(first, first + c["t"], device="cuda")
                scale[s["table"][i].long()[slot // c["page"]], :, slot % c["page"]] = step[i]
            out[name + "s"] = scale
        return out
    if op == "read":
        out = [torch.zeros((c["b"], c["ctx"], c["hk"], c["d"]), dtype=torch.float64, device="cuda") for _ in "kv"]
        for i, n in enumerate(_lens(c)):
            out[0][i, :n] = _exact_rows((ck, sk), s, c, i, 0, n)
            out[1][i, :n] = _exact_rows((cv, sv), s, c, i, 0, n)
        return out
    if op == "move":
        out = []
        for codes, scale in ((ck, sk), (cv, sv)):
            x = torch.empty((c["layers"], c["b"], c["t"], c["hk"], c["d"]), dtype=torch.float64, device="cuda")
            for i, first in enumerate(_lens(c)):
                to = [0] + s["path"][i, : _taken(c)[i]].tolist()
                to += range(len(to), c["t"])
                for layer in range(c["layers"]):
                    x[layer, i] = _exact_rows((codes[layer], scale[layer]), s, c, i, first, first + c["t"])[to]
            out.append(x)
        return out
    grp = c["hq"] // c["hk"]
    o = torch.zeros((c["b"], c["t"], c["hq"], c["d"]), dtype=torch.float64, device="cuda")
    for i, n in enumerate(_lens(c)):
        kk, vv = (_exact_rows(x, s, c, i, 0, n + c["t"]) for x in ((ck, sk), (cv, sv)))
        tree = torch.stack([(s["mask"][i] >> j) & 1 for j in range(c["t"])], 1) != 0  # [node, seen node]
        seen = torch.cat([tree.new_ones((c["t"], n)), tree], 1)
        for h in range(c["hq"]):
            z = s["q"][i, :, h].double() @ kk[:, h // grp].T * c["d"] ** -0.5
            o[i, :, h] = torch.softmax(torch.where(seen, z, -math.inf), -1) @ vv[:, h // grp]
    return o
