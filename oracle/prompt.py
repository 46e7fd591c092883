"""CPU oracle of the prompt's operators (causal attention over packed prompts, log probabilities), written from their
definitions in numpy, 64 bits."""
from __future__ import annotations

import numpy as np


def attention(q, k, v, offsets, scale):
    """q [N, Hq, D], k, v [N, Hk, D] -> (output, sum of |v| by weight, largest sum of |q k scale| of a row's products),
    each [N, Hq, D] or [N, Hq, 1]: the last two are what errors scale with.  Keys that a row does not see are not read."""
    q, k, v = (np.asarray(x, dtype=np.float64) for x in (q, k, v))
    grp = q.shape[1] // k.shape[1]
    out, size = np.zeros(q.shape), np.zeros(q.shape)
    prod = np.zeros((*q.shape[:2], 1))
    for first, last in zip(offsets[:-1], offsets[1:]):
        n = last - first
        if n <= 0:
            continue
        seen = np.tril(np.ones((n, n), dtype=bool))
        for h in range(q.shape[1]):
            qq, kk, vv = q[first:last, h], k[first:last, h // grp], v[first:last, h // grp]
            with np.errstate(invalid="ignore", over="ignore"):
                s = np.where(seen, qq @ kk.T * scale, -np.inf)
                p = np.where(seen, np.exp(s - s.max(-1, keepdims=True)), 0)
                p /= p.sum(-1, keepdims=True)
                if np.isfinite(vv).all():
                    out[first:last, h], size[first:last, h] = p @ vv, p @ np.abs(vv)
                else:  # (0 times a value that is not finite is not 0)
                    for i in range(n):
                        out[first + i, h] = p[i, :i + 1] @ vv[:i + 1]
                        size[first + i, h] = p[i, :i + 1] @ np.abs(vv[:i + 1])
                prod[first:last, h, 0] = np.where(seen, np.abs(qq) @ np.abs(kk).T * abs(scale), 0).max(-1)
    return out, size, prod


def logprobs(x, tokens, top):
    """(log p of the tokens, entropy, top log p, top tokens) of logits x [rows, V]."""
    x = np.asarray(x, dtype=np.float64)
    rows, v = x.shape
    lp = np.empty_like(x)
    for r in range(rows):
        m = x[r].max()
        if np.isnan(x[r]).any() or m == np.inf:
            lp[r] = np.nan
        elif m == -np.inf:
            lp[r] = -np.inf
        else:
            lp[r] = x[r] - m - np.log(np.exp(x[r] - m).sum())
    with np.errstate(invalid="ignore"):
        entropy = -np.where(lp == -np.inf, 0.0, np.exp(lp) * lp).sum(-1) + 0.0
    order = np.argsort(-x, axis=-1, kind="stable")[:, :top]
    given = (tokens >= 0) & (tokens < v)
    logp = np.where(given, lp[np.arange(rows), np.where(given, tokens, 0)], 0.0)
    bad = np.isnan(lp).any(-1, keepdims=True)
    return logp, entropy, np.take_along_axis(lp, order, -1), np.where(bad, -1, order)
