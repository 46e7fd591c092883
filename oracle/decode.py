"""CPU oracle of the speculative-decoding operators (rotary positions, paged int8 KV cache, tree attention, draft
verification), written from their definitions in numpy: 64 bits, except where the definition itself is a 32-bit one
(the quantiser's scale and quotient, the verifier's comparisons)."""
from __future__ import annotations

import numpy as np


def rotate(x, pos, freq, mag=1.0, interleaved=False):
    """x [.., heads, D], pos [..], freq [rot / 2] radians per position -> float64."""
    y = np.array(x, dtype=np.float64)
    ang = np.asarray(pos, dtype=np.float64)[..., None, None] * np.asarray(freq, dtype=np.float64)
    c, s, half = np.cos(ang) * mag, np.sin(ang) * mag, len(freq)
    i, j = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    a, b = y[..., i].copy(), y[..., j].copy()
    y[..., i], y[..., j] = a * c - b * s, a * s + b * c
    return y


def quantise(x):
    """x [.., D] float32 -> (codes int8, scale float32 [..]): scale = max|x| / 127 ignoring NaN, NaN quotient -> 0."""
    x = np.asarray(x, dtype=np.float32)
    with np.errstate(all="ignore"):
        s = (np.fmax.reduce(np.abs(x), axis=-1, initial=np.float32(0)) / np.float32(127)).astype(np.float32)
        q = np.clip(np.rint(x / s[..., None]), -127, 127)
    return np.where(np.isnan(q), 0, q).astype(np.int8), s


def slot(table, b, s, page, pages):
    """(page, row) of a slot, or None if it does not exist."""
    if s < 0 or s // page >= table.shape[1] or not 0 <= table[b, s // page] < pages:
        return None
    return int(table[b, s // page]), int(s % page)


def write(cache, table, start, k, v, counts=None):
    """Quantise float32 k, v [B, T, H, D] into cache = (k, v, ks, vs), in place."""
    pages, _, page, _ = cache[0].shape
    for b in range(k.shape[0]):
        for i in range(k.shape[1] if counts is None else min(k.shape[1], counts[b])):
            at = slot(table, b, int(start[b]) + i, page, pages)
            if at is None:
                continue
            for x, codes, scale in ((k, cache[0], cache[2]), (v, cache[1], cache[3])):
                codes[at[0], :, at[1]], scale[at[0], :, at[1]] = quantise(x[b, i])


def read(cache, table, start, n, lens=None):
    """float64 values [B, n, H, D] of k and v (one rounding away from the operator's)."""
    pages, h, page, d = cache[0].shape
    out = np.zeros((2, table.shape[0], n, h, d))
    for b in range(table.shape[0]):
        for i in range(n if lens is None else max(0, min(n, lens[b]))):
            at = slot(table, b, (0 if start is None else int(start[b])) + i, page, pages)
            if at is not None:
                for o, codes, scale in ((out[0], cache[0], cache[2]), (out[1], cache[1], cache[3])):
                    o[b, i] = codes[at[0], :, at[1]].astype(np.float64) * scale[at[0], :, at[1], None]
    return out


def move(cache, table, start, path, taken):
    """One layer's rows of accepted nodes to slots start + 1 ..; in place."""
    pages, _, page, _ = cache[0].shape
    t = path.shape[1]
    for b in range(table.shape[0]):
        todo = []
        for i in range(max(0, min(int(taken[b]), t - 1))):
            if not 0 <= path[b, i] < t:
                continue
            s = slot(table, b, int(start[b]) + int(path[b, i]), page, pages)
            d = slot(table, b, int(start[b]) + 1 + i, page, pages)
            if s is not None and d is not None:
                todo.append((d, [x[s[0], :, s[1]].copy() for x in cache]))
        for d, rows in todo:
            for x, r in zip(cache, rows):
                x[d[0], :, d[1]] = r


def tree_mask(parents):
    """[B, T] uint64 masks and depths from parents by following them."""
    bsz, t = parents.shape
    mask, depth = np.zeros((bsz, t), dtype=np.uint64), np.zeros((bsz, t), dtype=np.int64)
    for b in range(bsz):
        for i in range(t):
            seen, at = [], i
            while at != 0 and 0 <= parents[b, at] < at:
                seen.append(at)
                at = int(parents[b, at])
            if at == 0:
                for j in seen + [0]:
                    mask[b, i] |= np.uint64(1) << np.uint64(j)
                depth[b, i] = len(seen)
    return mask, depth


def attention(q, cache, table, ctx, mask=None, counts=None, scale=None):
    """q [B, T, Hq, D] -> (o, a, reach): the attention in float64, sum w |v| (what errors scale with) and the
    largest scale * sum |q| |k| of a visible key (what the scores' rounding scales with)."""
    bsz, t, hq, d = q.shape
    pages, h, page, _ = cache[0].shape
    scale = d ** -0.5 if scale is None else scale
    q = q.astype(np.float64)
    o, a, reach = np.zeros(q.shape), np.zeros(q.shape), 0.0
    for b in range(bsz):
        nodes = t if counts is None else max(0, min(t, int(counts[b])))
        c = max(0, int(ctx[b]))
        at = [(j, slot(table, b, j, page, pages)) for j in range(c + nodes)]
        at = [(j, x) for j, x in at if x is not None]
        if not at:
            continue
        pg, rw, js = (np.array(z) for z in ([x[0] for _, x in at], [x[1] for _, x in at], [j for j, _ in at]))
        k = cache[0][pg, :, rw].astype(np.float64) * cache[2][pg, :, rw].astype(np.float64)[..., None]
        v = cache[1][pg, :, rw].astype(np.float64) * cache[3][pg, :, rw].astype(np.float64)[..., None]
        for i in range(nodes):
            bits = ((1 << (i + 1)) - 1) if mask is None else int(np.uint64(mask[b, i]))
            see = np.array([int(j) < c or (bits >> (int(j) - c)) & 1 == 1 for j in js], dtype=bool)
            if not see.any():
                continue
            for x in range(hq):
                kk, vv = k[see, x // (hq // h)], v[see, x // (hq // h)]
                s = kk @ q[b, i, x] * scale
                top = s.max()
                if top == -np.inf:
                    continue
                w = np.exp(s - top)
                w /= w.sum()
                o[b, i, x], a[b, i, x] = w @ vv, w @ np.abs(vv)
                reach = max(reach, float((np.abs(kk) @ np.abs(q[b, i, x])).max()) * abs(scale))
    return o, a, reach


def verify(p, tokens, parents, u, e, draft=None):
    """The walk of one batch: (n [B], path [B, T], out [B, T])."""
    f = np.float32
    bsz, t, v = p.shape
    n, path, out = np.zeros(bsz, np.int32), np.full((bsz, t), -1, np.int32), np.full((bsz, t), -1, np.int64)
    for b in range(bsz):
        cur, w, z = 0, p[b, 0].astype(f), f(1)
        for i in range(1, t):
            if parents[b, i] != cur:
                continue
            x = int(tokens[b, i])
            if 0 <= x < v:
                qx = f(1) if draft is None else f(draft[b, cur, x])
                if f(f(u[b, i]) * qx) * z < w[x]:
                    path[b, n[b]], out[b, n[b]] = i, x
                    n[b] += 1
                    cur, w, z = i, p[b, i].astype(f), f(1)
                    continue
            if draft is not None:
                w = np.maximum(w - z * draft[b, cur].astype(f), f(0))
            elif 0 <= x < v:
                w = w.copy()
                w[x] = 0
            z = f(w.sum(dtype=np.float64))
        if not (w > 0).any():
            w = p[b, cur].astype(f)
        with np.errstate(all="ignore"):
            score = np.where(w > 0, w / e[b].astype(f), f(-1))
        out[b, n[b]] = int(np.argmax(score)) if (w > 0).any() else 0
    return n, path, out
