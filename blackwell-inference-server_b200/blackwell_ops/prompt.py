"""Operators of a prompt's pass, as hand-written sm_100a kernels: what a decoder computes on whole prompts, next to
``blackwell_ops.decode``, which has its steps (and the norms, the rotation and the cache's write for both).

* ``prompt_attention``: causal attention over packed prompts of different lengths, grouped query heads;
* ``token_logprobs``: log probabilities of given tokens, the distribution's entropy and its most likely tokens.

Packed prompts lie one behind the other in the first dimension: sequence b has the rows ``offsets[b]`` to
``offsets[b + 1]`` (int32 on the device, so a captured graph serves other lengths).

Kernels run on torch's current stream of the inputs' device; outputs come from the caching allocator and carry no
gradient.  Errors are ``RuntimeError``.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from ._lib import DTYPE_CODE, lib
from .decode import MAX_HEAD_DIM, _call, _new, _rows

MAX_TOP = 32  # alternatives of a token

_LOGITS = (torch.float16, torch.bfloat16, torch.float32)


def _tiled(x: torch.Tensor, n: int, heads: int, st: int, sh: int) -> tuple[torch.Tensor, int, int]:
    """x [n, heads, D], its strides of a row and a head; a copy unless its rows lie as the tensor-core kernel's copies
    want them: each on a 16-byte boundary, none twice."""
    if not (x.data_ptr() % 16 or st % 8 or sh % 8 or (st == 0 and n > 1) or (sh == 0 and heads > 1)):
        return x, st, sh
    x = x.clone(memory_format=torch.contiguous_format)
    return x, *x.stride()[-3:-1]


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor,
                     softmax_scale: float | None = None) -> torch.Tensor:
    """Causal attention over packed prompts: q [N, Hq, D], k and v [N, Hk, D] (fp16 or bf16) -> [N, Hq, D].

    Row i of a sequence sees the sequence's rows up to itself.  ``offsets`` [B + 1] int32, not descending; rows of no
    sequence (before ``offsets[0]``, behind ``offsets[B]``) give zeros.  Query head h reads key head
    ``h // (Hq / Hk)``.  ``softmax_scale`` defaults to ``D ** -0.5``.  A sequence's results do not depend on the others.
    Infinite and NaN elements of v go to that element of every row that sees them, whatever their weight.

    The tensor-core kernel takes D = 64 or 128, at most 128 query heads a key head and a positive scale (rows that do not
    start on 16-byte boundaries are copied first); other calls go to a plain kernel, a hundred times slower on long
    prompts."""
    if q.dim() != 3:
        raise RuntimeError("q must be [N, heads, D]")
    lead = q.shape[:-2]
    q, shape, _, n, _, qt, qh = _rows(q, "q", lead)
    k, kshape, _, _, _, kt, kh = _rows(k, "k", lead)
    v, vshape, _, _, _, vt, vh = _rows(v, "v", lead)
    dev, dt = q.device, q.dtype
    hq, d = shape[-2:]
    hk = kshape[-2]
    if k.dtype is not dt or v.dtype is not dt or k.device != dev or v.device != dev:
        raise RuntimeError("q, k and v must share one dtype and device")
    if kshape[-1] != d or vshape != kshape:
        raise RuntimeError("k and v must be [N, heads, D] of q's head dimension")
    if not 1 <= d <= MAX_HEAD_DIM:
        raise RuntimeError(f"the head dimension must be 1 to {MAX_HEAD_DIM}")
    if hq == 0 or hk == 0 or hq % hk:
        raise RuntimeError("q's heads must be a multiple of k's")
    if offsets.dtype is not torch.int32 or offsets.device != dev:
        raise RuntimeError("offsets must be int32 on the inputs' device")
    if offsets.dim() != 1 or offsets.shape[0] == 0:
        raise RuntimeError("offsets must be [B + 1]")
    offsets = offsets.contiguous()
    if d in (64, 128):
        q, qt, qh = _tiled(q, n, hq, qt, qh)
        k, kt, kh = _tiled(k, n, hk, kt, kh)
        v, vt, vh = _tiled(v, n, hk, vt, vh)
    out = _new(shape, dt, dev)
    _call("prompt_attention", dev, lib.bw_prompt_attention, q.data_ptr(), qt, qh, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh,
          DTYPE_CODE[dt], out.data_ptr(), offsets.data_ptr(), offsets.shape[0] - 1, n, hq, hk, d,
          d ** -0.5 if softmax_scale is None else float(softmax_scale))
    return out


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor      # [..] fp32
    entropy: torch.Tensor       # [..] fp32
    top_logprobs: torch.Tensor  # [.., top] fp32
    top_tokens: torch.Tensor    # [.., top] int64


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> TokenLogprobs:
    """Log probabilities of ``tokens`` [..] int64 under ``logits`` [.., V] (fp16, bf16 or fp32), the entropy of each
    distribution, and its ``top`` most likely tokens (at most 32 and V) with their log probabilities, in nats.

    A token outside [0, V) (padding) is not scored: 0.  Ties go to the lowest token.  Logits of -inf have no
    probability; a row of nothing else has entropy 0 and log probabilities of -inf.  A row with a NaN or +inf gives NaN,
    and tokens -1.  32-bit sums in one order: a row's results depend neither on the others nor on where it lies."""
    if not logits.is_cuda:
        raise RuntimeError("logits must be CUDA")
    if logits.dtype not in _LOGITS:
        raise RuntimeError("logits must be fp16, bf16 or fp32")
    if logits.dim() < 1 or logits.shape[-1] == 0:
        raise RuntimeError("logits must be [.., V]")
    dev, lead, v = logits.device, logits.shape[:-1], logits.shape[-1]
    if tokens.dtype is not torch.int64 or tokens.device != dev or tokens.shape != lead:
        raise RuntimeError(f"tokens must be int64 {list(lead)} on the logits' device")
    if not 0 <= top <= MAX_TOP:
        raise RuntimeError(f"top must be 0 to {MAX_TOP}")
    top = min(top, v)
    if logits.dim() != 2:
        logits = logits.reshape(-1, v)
    if logits.stride(1) != 1 and v > 1:
        logits = logits.contiguous()
    tokens = tokens.contiguous()
    rows = logits.shape[0]
    logp, entropy = _new((rows,), torch.float32, dev), _new((rows,), torch.float32, dev)
    top_logp, top_tok = _new((rows, top), torch.float32, dev), _new((rows, top), torch.int64, dev)
    _call("token_logprobs", dev, lib.bw_token_logprobs, logits.data_ptr(), DTYPE_CODE[logits.dtype], logits.stride(0),
          tokens.data_ptr(), rows, v, top, logp.data_ptr(), entropy.data_ptr(), top_logp.data_ptr(), top_tok.data_ptr())
    if len(lead) != 1:
        return TokenLogprobs(logp.view(lead), entropy.view(lead), top_logp.view(*lead, top), top_tok.view(*lead, top))
    return TokenLogprobs(logp, entropy, top_logp, top_tok)


__all__ = ["MAX_TOP", "TokenLogprobs", "prompt_attention", "token_logprobs"]
