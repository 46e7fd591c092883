"""Cases of the operators of a prompt's pass: norms of queries and keys for each head with the rotation (and the write
into the paged int8 KV cache) in the same pass, causal attention over whole packed prompts, and log probabilities of
given tokens with entropy and top alternatives.

Sizes are those of the decoders this repository already names (Qwen3-0.6B: 16 query / 8 key heads, vocabulary 151936;
Llama-3-8B: 32 / 8, vocabulary 128256; Llama-3-70B: 64 / 8; head dimension 128) and generic ones.

Conventions shared by every case: packed prompts lie one behind the other, sequence b's tokens at rows offsets[b] ..
offsets[b + 1], and rows behind the last one are the spare ones of a fixed-size batch.  Slot s of sequence b is row
s % page of page table[b, s // page] of the cache (int8 codes [pages, heads, page, D], one fp32 scale a token and head).
"""
import math
import sys

import torch

own = False

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}
BASE, EPS = 1000000.0, 1e-6


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step's queries and keys of a small batch: pure latency
        dict(name="norm rotary decode 16", op="norm", tokens=16, hq=16, hk=8, d=128, rot=128, layout="half",
             scaling="none", maxpos=4096, dt="bf16"),
        # a long prompt, frequencies scaled for long contexts
        dict(name="norm rotary prompt 8191", op="norm", tokens=8191, hq=32, hk=8, d=128, rot=128, layout="half",
             scaling="llama3", maxpos=131072, dt="bf16"),
        # one decode step of 64 sequences: normalised, turned and written into the cache, read back
        dict(name="norm write decode 64", op="write", b=64, t=1, packed=False, hq=32, hk=8, d=128, rot=128, page=16,
             ctx=4001, layout="half", scaling="none", dt="f16"),
        # a server's prompts of different lengths in one pass, keys kept for the prompts' own attention
        dict(name="norm write packed 8 x 1k", op="write", b=8, t=1023, packed=True, hq=16, hk=8, d=128, rot=128,
             page=64, ctx=0, layout="half", scaling="none", dt="bf16"),
        # one short prompt: latency
        dict(name="attention 1 x 17", op="attention", b=1, t=17, hq=16, hk=8, d=128, pad=0, dt="f16"),
        # a server's batch of ordinary prompts of different lengths, one slot of it idle
        dict(name="attention packed 24 x 1k", op="attention", b=24, t=1021, hq=32, hk=8, d=128, pad=7, dt="bf16"),
        # groups of seven query heads, head dimension 64
        dict(name="attention packed 6 x 2k, 28 / 4", op="attention", b=6, t=2050, hq=28, hk=4, d=64, pad=0, dt="f16"),
        # one very long prompt: bound by arithmetic
        dict(name="attention 1 x 16k", op="attention", b=1, t=16383, hq=16, hk=8, d=128, pad=0, dt="bf16"),
        # one sequence's next token with its twenty alternatives: latency
        dict(name="logprobs 1, top 20", op="logprobs", rows=1, v=151936, top=20, masked=0.0, dt="bf16"),
        # a decode step of 64 sequences, most tokens excluded by a grammar
        dict(name="logprobs 64, top 5", op="logprobs", rows=64, v=128256, top=5, masked=0.9, dt="f16"),
        # logits in 32 bits of an odd vocabulary
        dict(name="logprobs 333 odd, top 8", op="logprobs", rows=333, v=50257, top=8, masked=0.0, dt="f32"),
        # every token of a prompt scored, with the one that the model would have taken
        dict(name="logprobs prompt 2047", op="logprobs", rows=2047, v=151936, top=1, masked=0.0, dt="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw(rng):
    op = rng.choice(["norm", "write", "attention", "attention", "logprobs", "logprobs"])
    dt = rng.choice(["f16", "bf16"])
    hq, hk = rng.choice([(16, 8), (32, 8), (64, 8), (8, 8), (28, 4), (12, 1)])
    d = rng.choice([64, 128])
    layout, scaling, rot = rng.choice(["half", "interleaved"]), rng.choice(["none", "llama3"]), rng.choice([d, d, d // 2])
    if op == "norm":
        return dict(op=op, tokens=_log(rng, 1, 8191), hq=hq, hk=hk, d=d, rot=rot, layout=layout, scaling=scaling,
                    maxpos=_log(rng, 1024, 131072), dt=dt)
    if op == "write":
        b = _log(rng, 1, 64)
        return dict(op=op, b=b, t=_log(rng, 1, max(1, 8192 // b)), packed=rng.random() < 0.6, hq=hq, hk=hk, d=d, rot=rot,
                    page=rng.choice([16, 32, 64, 128]), ctx=rng.choice([0, _log(rng, 1, 4096)]), layout=layout,
                    scaling=scaling, dt=dt)
    if op == "attention":
        return dict(op=op, b=_log(rng, 1, 64), t=_log(rng, 1, 16383), hq=hq, hk=hk, d=d, pad=rng.choice([0, rng.randint(1, 40)]),
                    dt=dt)
    v = rng.choice([32000, 50257, 128256, 151936, _log(rng, 100, 151936)])
    return dict(op=op, rows=_log(rng, 1, 4096), v=v, top=rng.choice([0, 1, rng.randint(2, 32)]),
                masked=rng.choice([0.0, 0.5, 0.99]), dt=rng.choice(["f16", "bf16", "f32"]))


def draw(rng):
    while True:
        c = _draw(rng)
        if c["op"] == "attention":  # the plain form holds every score
            if work(c)["flops"] <= 1.1e12 and c["b"] * c["t"] ** 2 * c["hq"] <= 4.3e9 and c["b"] * c["t"] <= 32768:
                return c
        elif c["op"] == "logprobs":
            if c["rows"] * c["v"] <= 3.11e8:
                return c
        elif work(c)["bytes"] <= 340e6 and (c["op"] == "norm" or c["b"] * (c["ctx"] + c["t"]) * c["hk"] * c["d"] <= 6.0e8):
            return c


def _lens(c):
    """Lengths of a batch: from all of t down to a b-th of it, the last of eight and more an idle slot."""
    n = [max(1, c["t"] - c["t"] * i // c["b"]) for i in range(c["b"])]
    if c["b"] >= 8:
        n[-1] = 0
    return n


def _total(c):
    return sum(_lens(c)) if c.get("packed", True) else c["b"] * c["t"]


def work(c):
    op, e = c["op"], 4 if c["dt"] == "f32" else 2
    if op == "norm":
        n = c["tokens"] * (c["hq"] + c["hk"]) * c["d"]
        return {"bytes": 2 * e * n + 4 * c["tokens"], "flops": 6 * n}
    if op == "write":  # 16-bit rows in, queries (and packed prompts' keys) out, codes and scales written and read back as values
        n = _total(c)
        q, kv = n * c["hq"] * c["d"], n * c["hk"] * c["d"]
        return {"bytes": 2 * e * q + kv * (2 * e + (e if c["packed"] else 0) + 2 + 2 * e) + 8 * n * c["hk"],
                "flops": 6 * (q + kv) + 4 * kv}
    if op == "attention":
        pairs = sum(n * (n + 1) // 2 for n in _lens(c))
        return {"bytes": 2 * e * _total(c) * (c["hq"] + c["hk"]) * c["d"], "flops": 4 * c["hq"] * c["d"] * pairs}
    n = c["rows"] * c["v"]
    return {"bytes": e * n + c["rows"] * (16 + 12 * c["top"]), "flops": 5 * n}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + 29)


def _normal(g, shape, dt):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dt)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _frequencies(c):
    """Radians per position of each turned pair (64-bit floats)."""
    f = BASE ** (-torch.arange(c["rot"] // 2, dtype=torch.float64) * 2.0 / c["rot"])
    if c["scaling"] == "none":
        return f
    turns = LLAMA3["original_max_position_embeddings"] * f / (2 * math.pi)
    lo, hi = LLAMA3["low_freq_factor"], LLAMA3["high_freq_factor"]
    mix = ((turns - lo) / (hi - lo)).clamp(0, 1)
    return f * ((1 - mix) / LLAMA3["factor"] + mix)


def _decode():
    if "blackwell-inference-server_b200" not in sys.path:
        sys.path.insert(1, "blackwell-inference-server_b200")
    import blackwell_ops.decode as ops
    return ops


def _prompt():
    _decode()
    import blackwell_ops.prompt as ops
    return ops


def prepare(c, seed):
    g, op, dt = _gen(seed), c["op"], DT[c["dt"]]
    s = {"c": c}
    if op == "logprobs":
        # a model's logits: wide, with a few likely tokens; what a grammar excludes is -inf
        x = torch.empty((c["rows"], c["v"]), device="cuda").normal_(generator=g).mul_(2.5)
        likely = torch.randint(0, c["v"], (c["rows"], 6), generator=g, device="cuda")
        x.scatter_add_(1, likely, torch.rand((c["rows"], 6), generator=g, device="cuda") * 12)
        if c["masked"]:
            x.masked_fill_(torch.rand(x.shape, generator=g, device="cuda") < c["masked"], -math.inf)
        s["logits"] = x.to(dt)
        # most given tokens are likely ones, some any, one in eight is padding that is not scored
        pick = torch.rand((c["rows"],), generator=g, device="cuda")
        tok = torch.where(pick < 0.7, likely[:, 0], torch.randint(0, c["v"], (c["rows"],), generator=g, device="cuda"))
        s["tokens"] = torch.where(pick > 0.875, -100, tok)
        return s
    if op in ("norm", "write"):
        # the norms' weights of a trained model spread around one
        s["wq"], s["wk"] = ((1 + 0.3 * _normal(g, (c["d"],), torch.float32)).to(dt) for _ in "qk")
        s["freq"] = _frequencies(c).cuda()
        if own:
            s["plan"] = _decode().rotary_plan(c["rot"], base=BASE, scaling=LLAMA3 if c["scaling"] == "llama3" else None,
                                              interleaved=c["layout"] == "interleaved", device="cuda")
    if op == "norm":
        # queries and keys lie side by side with the values, as one projection leaves them
        s["qkv"] = 3 * _normal(g, (c["tokens"], c["hq"] + 2 * c["hk"], c["d"]), dt)
        s["pos"] = torch.randint(0, c["maxpos"], (c["tokens"],), generator=g, device="cuda", dtype=torch.int32)
        return s
    lens = _lens(c)
    s["offsets"] = _i32([sum(lens[:i]) for i in range(c["b"] + 1)])
    if op == "attention":
        n = _total(c) + c["pad"]
        s["q"], s["k"] = 2.5 * _normal(g, (n, c["hq"], c["d"]), dt), _normal(g, (n, c["hk"], c["d"]), dt)
        # the values are a part of the projection's output
        s["v"] = _normal(g, (n, 2 * c["hk"], c["d"]), dt)[:, c["hk"]:]
        return s
    # the cache's pages are scattered as a server's allocator leaves them
    per = -(-(c["ctx"] + c["t"]) // c["page"])
    pages = c["b"] * per + 3
    s["table"] = torch.randperm(pages, generator=g, device="cuda")[: c["b"] * per].to(torch.int32).view(c["b"], per)
    shape = (pages, c["hk"], c["page"], c["d"])
    s["cache"] = [torch.zeros(shape, dtype=torch.int8, device="cuda") for _ in "kv"]
    s["cache"] += [torch.zeros(shape[:-1], dtype=torch.float32, device="cuda") for _ in "kv"]
    s["start"] = _i32([c["ctx"] - c["ctx"] // 2 * i // c["b"] for i in range(c["b"])])
    s["lens"] = _i32(lens if c["packed"] else [c["t"]] * c["b"])
    h = c["hq"] + 2 * c["hk"]
    s["qkv"] = 3 * _normal(g, (_total(c), h, c["d"]) if c["packed"] else (c["b"], c["t"], h, c["d"]), dt)
    if c["packed"]:
        seq, at = _places(s, _total(c))
        s["pos"] = s["start"][seq] + at.to(torch.int32)
    else:
        s["pos"] = s["start"][:, None] + torch.arange(c["t"], device="cuda", dtype=torch.int32)
    if own:
        s["kv"] = _decode().KVCacheInt8(*s["cache"])
    return s


def _places(s, n):
    """Sequence and place in it of n packed rows."""
    row = torch.arange(n, device="cuda")
    seq = torch.searchsorted(s["offsets"].long(), row, right=True) - 1
    seq = seq.clamp(max=s["offsets"].shape[0] - 2)
    return seq, row - s["offsets"].long()[seq]


# ------------------------------------------------------------------ the framework's calls and the plain forms
def run(s):
    return (_own if own else _plain)(s, s["c"])


def _own(s, c):
    op = c["op"]
    if op == "logprobs":
        return list(_prompt().token_logprobs(s["logits"], s["tokens"], top=c["top"]))
    if op == "attention":
        return _prompt().prompt_attention(s["q"], s["k"], s["v"], s["offsets"])
    ops = _decode()
    q, k, v = s["qkv"].split([c["hq"], c["hk"], c["hk"]], dim=-2)
    if op == "norm":
        return list(ops.norm_rotary(q, k, s["pos"], s["plan"], s["wq"], s["wk"], eps=EPS))
    q, k = ops.norm_rotary_kv_write_int8(q, k, v, s["pos"], s["plan"], s["kv"], s["table"], s["start"], s["wq"], s["wk"],
                                         eps=EPS, offsets=s["offsets"] if c["packed"] else None, keys=c["packed"])
    out = {"q": q, "k": k} if c["packed"] else {"q": q}
    out["cache k"], out["cache v"] = ops.kv_read_int8(s["kv"], s["table"], s["start"], c["t"], lens=s["lens"],
                                                      dtype=DT[c["dt"]])
    out["ks"], out["vs"] = s["cache"][2:]
    return out


def _normed(x, w):
    x = x.float()
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()


def _turn(x, pos, s, c):
    """The rotation in 32 bits (angles in 64); x [.., heads, D], pos [..]."""
    a = pos.double()[..., None, None] * s["freq"]
    co, si = torch.cos(a).float(), torch.sin(a).float()
    r = c["rot"]
    if c["layout"] == "half":
        x1, x2 = x[..., : r // 2], x[..., r // 2 : r]
        y = torch.cat([x1 * co - x2 * si, x1 * si + x2 * co], -1)
    else:
        x1, x2 = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack([x1 * co - x2 * si, x1 * si + x2 * co], -1).flatten(-2)
    return torch.cat([y, x[..., r:]], -1)


def _plain(s, c):
    op, dt = c["op"], DT[c["dt"]]
    if op == "logprobs":
        return _plain_logprobs(s, c)
    if op == "attention":
        return _plain_attention(s, c)
    q, k, v = s["qkv"].split([c["hq"], c["hk"], c["hk"]], dim=-2)
    q, k = _turn(_normed(q, s["wq"]), s["pos"], s, c), _turn(_normed(k, s["wk"]), s["pos"], s, c)
    if op == "norm":
        return [q.to(dt), k.to(dt)]
    out = {"q": q.to(dt), "k": k.to(dt)} if c["packed"] else {"q": q.to(dt)}
    t = torch.arange(c["t"], device="cuda")
    if c["packed"]:
        seq, at = _places(s, _total(c))
    else:
        seq, at = torch.arange(c["b"], device="cuda")[:, None], t
    slot = s["start"].long()[seq] + at
    page, row = s["table"].long()[seq, slot // c["page"]], slot % c["page"]
    _store(k, s["cache"][0], s["cache"][2], page, row)
    _store(v.float(), s["cache"][1], s["cache"][3], page, row)
    # the written slots read back as values, zeros behind a sequence's last
    slot = s["start"].long()[:, None] + t
    page, row = s["table"].long().gather(1, slot // c["page"]), slot % c["page"]
    keep = (t < s["lens"][:, None])[..., None, None]
    out["cache k"] = _values(s["cache"][0], s["cache"][2], page, row, keep).to(dt)
    out["cache v"] = _values(s["cache"][1], s["cache"][3], page, row, keep).to(dt)
    out["ks"], out["vs"] = s["cache"][2:]
    return out


def _store(x, codes, scale, page, row):
    sc = x.abs().amax(-1) / 127
    codes[page, :, row, :] = torch.round(x / sc[..., None]).clamp(-127, 127).to(torch.int8)
    scale[page, :, row] = sc


def _values(codes, scale, page, row, keep):
    return torch.where(keep, codes[page, :, row].float() * scale[page, :, row][..., None], 0.0)


def _plain_attention(s, c):
    """Sequences padded to the longest, every score held."""
    b, t, hk, d, grp = c["b"], c["t"], c["hk"], c["d"], c["hq"] // c["hk"]
    n = s["q"].shape[0]
    at = torch.arange(t, device="cuda")
    rows = (s["offsets"].long()[:-1, None] + at).clamp(max=n - 1)  # [b, t]
    q = s["q"].float()[rows].view(b, t, hk, grp, d).permute(0, 2, 3, 1, 4).reshape(b, hk, grp * t, d)
    k, v = s["k"].float()[rows].permute(0, 2, 3, 1), s["v"].float()[rows].permute(0, 2, 1, 3)
    w = torch.matmul(q, k).view(b, hk, grp, t, t).mul_(1 / math.sqrt(d))
    w.masked_fill_(at[None, :] > at[:, None], -math.inf)
    w.sub_(w.amax(-1, keepdim=True)).exp_()
    total = w.sum(-1)
    o = torch.matmul(w.view(b, hk, grp * t, t), v).view(b, hk, grp, t, d) / total[..., None]
    o = o.permute(0, 3, 1, 2, 4).reshape(b, t, c["hq"], d)
    seq, place = _places(s, n)
    real = (torch.arange(n, device="cuda") < s["offsets"][-1])[:, None, None]
    return torch.where(real, o[seq, place.clamp(max=t - 1)], 0.0).to(s["q"].dtype)


def _plain_logprobs(s, c):
    """What is excluded has no weight; a row that excludes everything has no entropy, and its tokens are impossible."""
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    z = x - top
    w = torch.exp(z)
    total = w.sum(-1, dtype=torch.float64)
    lead = torch.where(z == -math.inf, 0.0, z * w).sum(-1, dtype=torch.float64)
    some = total > 0
    norm = torch.where(some, torch.log(total), 0.0)
    entropy = torch.where(some, norm - lead / torch.where(some, total, 1.0), 0.0).float()
    given = (s["tokens"] >= 0) & (s["tokens"] < c["v"])
    logp = z.gather(1, s["tokens"].clamp(0, c["v"] - 1)[:, None])[:, 0] - norm
    logp = torch.where(given, logp, 0.0).float()
    out = [logp, entropy]
    best, index = torch.sort(z, dim=-1, descending=True, stable=True)
    k = min(c["top"], c["v"])
    return out + [(best[:, :k] - norm[:, None]).float(), index[:, :k].contiguous()]


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_rows(x, w, pos, s, c):
    x = x.double()
    x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / c["d"] + EPS) * w.double()
    ang = pos.double()[..., None, None] * s["freq"]
    unit = torch.polar(torch.ones_like(ang), ang)
    r, y = c["rot"], x.clone()
    first = slice(0, r // 2) if c["layout"] == "half" else slice(0, r, 2)
    second = slice(r // 2, r) if c["layout"] == "half" else slice(1, r, 2)
    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * unit
    y[..., first], y[..., second] = z.real, z.imag
    return y


def exact(c, seed):
    op, s = c["op"], prepare(c, seed)
    if op == "logprobs":
        return _exact_logprobs(s, c)
    if op == "attention":
        return _exact_attention(s, c)
    hq, hk = c["hq"], c["hk"]
    q = _exact_rows(s["qkv"][..., :hq, :], s["wq"], s["pos"], s, c)
    k = _exact_rows(s["qkv"][..., hq : hq + hk, :], s["wk"], s["pos"], s, c)
    if op == "norm":
        return [q, k]
    v = s["qkv"][..., hq + hk :, :].double()
    out = {"q": q, "k": k} if c["packed"] else {"q": q}
    scales = []
    for name, x, scale in (("cache k", k, s["cache"][2].double()), ("cache v", v, s["cache"][3].double())):
        step = x.abs().max(-1).values / 127
        codes = torch.round(x / step[..., None]) * step[..., None]
        back = torch.zeros((c["b"], c["t"], hk, c["d"]), dtype=torch.float64, device="cuda")
        for i in range(c["b"]):
            n, first, a = int(s["lens"][i]), int(s["start"][i]), int(s["offsets"][i])
            mine, m = (codes[a : a + n], step[a : a + n]) if c["packed"] else (codes[i], step[i])
            back[i, :n] = mine
            slot = torch.arange(first, first + n, device="cuda")
            scale[s["table"][i].long()[slot // c["page"]], :, slot % c["page"]] = m
        out[name] = back
        scales.append(scale)
    out["ks"], out["vs"] = scales
    return out


def _exact_attention(s, c):
    grp, o = c["hq"] // c["hk"], torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for n in _lens(c):
        for h in range(c["hq"]):
            z = s["q"][first : first + n, h].double() @ s["k"][first : first + n, h // grp].double().T * c["d"] ** -0.5
            z = z.tril() + torch.full_like(z, -math.inf).triu(1)
            o[first : first + n, h] = torch.softmax(z, -1) @ s["v"][first : first + n, h // grp].double()
        first += n
    return o


def _exact_logprobs(s, c):
    k = min(c["top"], c["v"])
    out = [[], [], [], []]
    for row, token in zip(s["logits"], s["tokens"].tolist()):
        x = row.double()
        lp = x - torch.logsumexp(x, 0) if bool((x > -math.inf).any()) else x
        p = torch.exp(lp)
        out[0].append(lp[token] if 0 <= token < c["v"] else torch.zeros_like(lp[0]))
        out[1].append(-torch.where(p > 0, p * lp, 0.0).sum())
        order = torch.argsort(-x, stable=True)[:k]
        out[2].append(lp[order])
        out[3].append(order)
    return [torch.stack(x) for x in out]
