"""Speculative decoding over a paged int8 KV cache, as hand-written sm_100a kernels.

The operators of one decoder step next to the W8A16 linears:

* ``rotary`` turns queries and keys by their positions (``rotary_plan``: half or interleaved pairs,
  part of the head, frequencies scaled for long contexts); ``norm_rotary`` normalises each of their heads first,
  in the same pass;
* ``KVCacheInt8`` holds int8 codes and one fp32 scale per token and head in pages;
  ``kv_write_int8`` quantises new keys and values as they are written, ``rotary_kv_write_int8``
  rotates and writes in one launch (``norm_rotary_kv_write_int8``: normalises too, and takes packed
  sequences of different lengths), ``kv_read_int8`` gives values back, ``kv_move_int8`` moves the
  accepted nodes of a draft tree to their final slots in every layer;
* ``tree_attention_int8`` attends from the nodes of a draft tree (or one new token) to the cache;
  ``tree_positions`` gives a tree's masks and positions;
* ``verify_tree`` accepts drafted tokens against the target's probabilities from given random numbers.

Slot s of sequence b is row ``s % page`` of page ``table[b, s // page]``.  A slot past the table, or
whose entry is no page of the cache, does not exist: it is not written, reads as zero and is not seen.

Kernels run on torch's current stream of the inputs' device; outputs come from the caching allocator.
Errors are ``RuntimeError``.  The attention keeps a workspace per (device, stream), and one for each CUDA
graph that it is captured into, whose replays need no warm-up call and may run on any stream.
"""
from __future__ import annotations

import functools
import math

import torch

from ._lib import DTYPE_CODE, check, lib
from ._workspace import Workspaces

MAX_NODES = 64      # nodes of a draft tree: one bit each
MAX_HEAD_DIM = 256

_HALF = (torch.float16, torch.bfloat16)
_workspaces = Workspaces(zeroed=4096)  # the tickets, in a prefix of one size for every shape


# These operators are called once a layer and step, so what a call costs on the host counts: the current
# stream's handle and device come without the objects around them.  The calls are torch's own, without a
# promise to stay; where one is missing the public call does the same (an attention call then takes 17.2 us
# on the host instead of 11.1).
try:
    from torch._C import _cuda_getCurrentRawStream as _stream
    from torch._C import _cuda_getDevice as _current_device
except ImportError:
    def _stream(index: int) -> int:
        return torch.cuda.current_stream(index).cuda_stream

    def _current_device() -> int:
        return torch.cuda.current_device()

try:  # the allocation that the compiler's generated code calls: 0.8 us where torch.empty takes 3
    from torch._C._dynamo.guards import _empty_strided_cuda as _empty_strided
except ImportError:
    _empty_strided = None


def _new(shape: tuple, dtype: torch.dtype, dev: torch.device) -> torch.Tensor:
    """A contiguous tensor."""
    n = len(shape)
    if _empty_strided is None or n > 4 or dev.index != _current_device():
        return torch.empty(shape, dtype=dtype, device=dev)
    if n == 4:
        a, b, c, d = shape
        return _empty_strided((a, b, c, d), (b * c * d, c * d, d, 1), dtype)
    if n == 3:
        a, b, c = shape
        return _empty_strided((a, b, c), (b * c, c, 1), dtype)
    return _empty_strided(tuple(shape), (shape[1], 1) if n == 2 else (1,), dtype)


def _call(op: str, dev: torch.device, fn, *args) -> None:
    """fn(*args, stream) on dev's current stream."""
    index = dev.index
    if index == _current_device():
        status = fn(*args, _stream(index))
    else:
        with torch.cuda.device(dev):
            status = fn(*args, _stream(index))
    if status:
        check(status, op)


def reset_workspaces() -> None:
    """Zero every cached attention workspace (needed only after a device-side timeout)."""
    _workspaces.reset()


@functools.lru_cache(maxsize=4096)
def _attention_bytes(index: int, b: int, t: int, hq: int, heads: int, d: int) -> int:
    with torch.cuda.device(index):
        return lib.bw_tree_attention_int8_workspace_size(b, t, hq, heads, d)


def _workspace(dev: torch.device, nbytes: int) -> torch.Tensor:
    """Scratch of the current stream; its tickets start, and stay, zero."""
    return _workspaces.get(dev, _stream(dev.index), nbytes)


# ---------------------------------------------------------------- rotary positions
def rotary_frequencies(rot_dim: int, base: float | None = None, scaling: dict | None = None) -> tuple[torch.Tensor, float]:
    """Radians per position of the ``rot_dim / 2`` pairs (float64, CPU) and the magnitude of a turned pair.

    ``base`` defaults to the ``rope_theta`` of ``scaling``, or 10000.  ``scaling`` is a Hugging Face ``rope_scaling`` / ``rope_parameters`` mapping:
    ``rope_type`` (or ``type``) one of

    * ``default``;
    * ``linear``: ``f / factor``;
    * ``ntk``: the base grows to ``base * factor ** (rot_dim / (rot_dim - 2))``;
    * ``llama3``: wavelengths over ``original_max_position_embeddings / low_freq_factor`` are stretched by
      ``factor``, those under ``.. / high_freq_factor`` kept, the ones between mixed linearly in their frequency;
    * ``yarn``: pairs that turn fewer than ``beta_slow`` times over the original context are stretched by
      ``factor``, those that turn more than ``beta_fast`` times kept, a linear ramp over the pairs between (whose
      ends are rounded outwards to whole pairs unless ``truncate`` is false); the magnitude is
      ``attention_factor``, or ``g(mscale) / g(mscale_all_dim)`` where both are given (and not 0), or ``g(1)``, with ``g(m) = 0.1 m ln(factor) + 1`` (1 for a factor of at most 1).
    """
    if rot_dim < 2 or rot_dim % 2:
        raise RuntimeError("rotary: rot_dim must be even and positive")
    scaling = scaling or {}
    if base is None:
        base = float(scaling.get("rope_theta") or 10000.0)
    if not (math.isfinite(base) and base > 1):
        raise RuntimeError("rotary: base must be over 1")
    kind = scaling.get("rope_type", scaling.get("type", "default")) or "default"
    i = torch.arange(rot_dim // 2, dtype=torch.float64)
    f = base ** (-2.0 * i / rot_dim)
    if kind == "default":
        return f, 1.0
    try:
        factor = float(scaling["factor"])
        if not (math.isfinite(factor) and factor > 0):
            raise RuntimeError("rotary: factor must be positive")
        if kind == "linear":
            return f / factor, 1.0
        if kind == "ntk":
            if rot_dim == 2:
                return f, 1.0
            return (base * factor ** (rot_dim / (rot_dim - 2))) ** (-2.0 * i / rot_dim), 1.0
        if kind == "llama3":
            lo, hi = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
            if not hi > lo:
                raise RuntimeError("rotary: high_freq_factor must be over low_freq_factor")
            turns = float(scaling["original_max_position_embeddings"]) * f / (2 * math.pi)
            keep = ((turns - lo) / (hi - lo)).clamp(0.0, 1.0)
            return keep * f + (1 - keep) * f / factor, 1.0
        if kind == "yarn":
            old = float(scaling["original_max_position_embeddings"])

            def pair_that_turns(n: float) -> float:
                return rot_dim * math.log(old / (n * 2 * math.pi)) / (2 * math.log(base))

            lo = pair_that_turns(float(scaling.get("beta_fast") or 32.0))
            hi = pair_that_turns(float(scaling.get("beta_slow") or 1.0))
            if scaling.get("truncate", True):
                lo, hi = math.floor(lo), math.ceil(hi)
            lo, hi = max(lo, 0), min(hi, rot_dim - 1)
            stretch = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
            mag = scaling.get("attention_factor")
            if mag is None:
                def grown(m: float) -> float:
                    return 0.1 * m * math.log(factor) + 1.0 if factor > 1 else 1.0

                both = scaling.get("mscale"), scaling.get("mscale_all_dim")
                mag = grown(float(both[0])) / grown(float(both[1])) if all(both) else grown(1.0)
            return stretch * f / factor + (1 - stretch) * f, float(mag)
    except KeyError as e:
        raise RuntimeError(f"rotary: {kind} scaling needs {e.args[0]}") from None
    raise RuntimeError(f"rotary: unknown scaling {kind!r}")


class RotaryPlan:
    """Frequencies of a rotation on one device: ``steps`` [rot_dim / 2] int64, turns per position in units of
    2^-64 (exact modulo one turn for every position), and the magnitude of a turned pair."""

    __slots__ = ("rot_dim", "interleaved", "magnitude", "steps", "device", "_ptr")

    def __init__(self, frequencies: torch.Tensor, magnitude: float = 1.0, interleaved: bool = False, device="cuda"):
        f = frequencies.detach().to("cpu", torch.float64).flatten()
        if not torch.isfinite(f).all() or not math.isfinite(magnitude):
            raise RuntimeError("rotary: frequencies and magnitude must be finite")
        steps = [round(x / (2 * math.pi) * 2.0**64) % 2**64 for x in f.tolist()]
        self.steps = torch.tensor([s - 2**64 if s >= 2**63 else s for s in steps], dtype=torch.int64).to(device)
        if not self.steps.is_cuda:
            raise RuntimeError("rotary: the plan must be on a CUDA device")
        self.device = self.steps.device
        self.rot_dim = 2 * f.numel()
        self.interleaved = bool(interleaved)
        self.magnitude = float(magnitude)
        self._ptr = self.steps.data_ptr()


def rotary_plan(rot_dim: int, base: float | None = None, scaling: dict | None = None, interleaved: bool = False,
                device="cuda") -> RotaryPlan:
    """A plan for ``rotary``: see ``rotary_frequencies`` for the arguments."""
    f, mag = rotary_frequencies(rot_dim, base, scaling)
    return RotaryPlan(f, mag, interleaved, device)


def _rows(x: torch.Tensor, name: str, lead: tuple) -> tuple[torch.Tensor, tuple, int, int, int, int, int]:
    """x [.., heads, d] as (x, shape, b, t, stride b, stride t, stride of heads); its leading dimensions are
    merged into two."""
    if not x.is_cuda:
        raise RuntimeError(f"{name} must be CUDA")
    if x.dtype not in _HALF:
        raise RuntimeError(f"{name} must be fp16 or bf16")
    shape = x.shape
    n = len(shape)
    if n < 3:
        raise RuntimeError(f"{name} must be [.., heads, d]")
    if shape[:-2] != lead:
        raise RuntimeError(f"{name} must have leading dimensions {list(lead)}")
    stride = x.stride()
    if stride[-1] != 1 and shape[-1] > 1:
        x = x.contiguous()
        stride = x.stride()
    if n == 4:
        return x, shape, shape[0], shape[1], stride[0], stride[1], stride[2]
    if n == 3:
        return x, shape, 1, shape[0], 0, stride[0], stride[1]
    x = x.reshape(-1, *shape[-3:])
    stride = x.stride()
    return x, shape, x.shape[0], x.shape[1], stride[0], stride[1], stride[2]


def _positions(positions: torch.Tensor, lead: tuple, dev: torch.device) -> torch.Tensor:
    if positions.device != dev:
        raise RuntimeError("positions must be on the inputs' device")
    if positions.dtype is not torch.int32 and positions.dtype is not torch.int64:
        raise RuntimeError("positions must be int32 or int64")
    if positions.shape != lead:
        raise RuntimeError(f"positions must be {list(lead)}")
    return positions if positions.is_contiguous() else positions.contiguous()


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor,
           plan: RotaryPlan) -> tuple[torch.Tensor, torch.Tensor | None]:
    """q [.., Hq, D] and k [.., Hk, D] (fp16 or bf16, or no k) turned by ``positions`` [..] (int32 or int64).

    Pair i of the first ``plan.rot_dim`` elements of a head turns by ``position * f_i``; the other
    elements are copied.  32-bit arithmetic, rounded once.  Returns new contiguous tensors."""
    lead = q.shape[:-2]
    q, shape, b, t, qb, qt, qh = _rows(q, "q", lead)
    dev, dt, hq, d = q.device, q.dtype, shape[-2], shape[-1]
    if plan.rot_dim > d or d > MAX_HEAD_DIM:
        raise RuntimeError(f"rotary: need rot_dim <= D <= {MAX_HEAD_DIM}")
    if plan.device != dev:
        raise RuntimeError("rotary: the plan is on another device")
    positions = _positions(positions, lead, dev)
    q_out = _new(shape, dt, dev)
    k_out, hk, kb, kt, kh, kp, kop = None, 0, 0, 0, 0, None, None
    if k is not None:
        k, kshape, _, _, kb, kt, kh = _rows(k, "k", lead)
        if k.dtype is not dt or k.device != dev or kshape[-1] != d:
            raise RuntimeError("k must have q's dtype, device and head dimension")
        hk = kshape[-2]
        k_out = _new(kshape, dt, dev)
        kp, kop = k.data_ptr(), k_out.data_ptr()
    if d:
        _call("rotary", dev, lib.bw_rotary, q.data_ptr(), qb, qt, qh, hq, kp, kb, kt, kh, hk, q_out.data_ptr(), kop,
              DTYPE_CODE[dt], b, t, d, positions.data_ptr(), positions.dtype is torch.int64, plan._ptr,
              plan.magnitude, plan.rot_dim, plan.interleaved)
    return q_out, k_out


def _weight(w: torch.Tensor | None, name: str, d: int, dt: torch.dtype, dev: torch.device) -> torch.Tensor | None:
    """A norm's contiguous weights [d], or none."""
    if w is None:
        return None
    if w.dtype is not dt or w.device != dev or w.shape != (d,):
        raise RuntimeError(f"{name} must be [{d}] of the inputs' dtype and device")
    return w if w.is_contiguous() else w.contiguous()


def norm_rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, plan: RotaryPlan,
                q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor | None]:
    """``rotary`` of queries and keys whose heads are normalised first, in one pass: each head's row x [D] becomes
    ``w * x / sqrt(mean(x^2) + eps)`` with w = ``q_weight`` or ``k_weight`` [D] (None: its rows are only turned).

    32-bit arithmetic, rounded once, behind the rotation.  The sum of squares is 32-bit, too: a bf16 row where it passes
    the range (values from 1.6e18 on, for D = 128) gives zeros, and with ``eps`` 0 one of values under 1e-19 is undefined.
    Returns new contiguous tensors."""
    lead = q.shape[:-2]
    q, shape, b, t, qb, qt, qh = _rows(q, "q", lead)
    dev, dt, hq, d = q.device, q.dtype, shape[-2], shape[-1]
    if plan.rot_dim > d or d > MAX_HEAD_DIM:
        raise RuntimeError(f"norm_rotary: need rot_dim <= D <= {MAX_HEAD_DIM}")
    if plan.device != dev:
        raise RuntimeError("norm_rotary: the plan is on another device")
    if not eps >= 0:
        raise RuntimeError("norm_rotary: eps must not be negative")
    positions = _positions(positions, lead, dev)
    q_weight, k_weight = _weight(q_weight, "q_weight", d, dt, dev), _weight(k_weight, "k_weight", d, dt, dev)
    q_out = _new(shape, dt, dev)
    k_out, hk, kb, kt, kh, kp, kop = None, 0, 0, 0, 0, None, None
    if k is not None:
        k, kshape, _, _, kb, kt, kh = _rows(k, "k", lead)
        if k.dtype is not dt or k.device != dev or kshape[-1] != d:
            raise RuntimeError("k must have q's dtype, device and head dimension")
        hk = kshape[-2]
        k_out = _new(kshape, dt, dev)
        kp, kop = k.data_ptr(), k_out.data_ptr()
    _call("norm_rotary", dev, lib.bw_norm_rotary, q.data_ptr(), qb, qt, qh, hq, kp, kb, kt, kh, hk, q_out.data_ptr(), kop,
          DTYPE_CODE[dt], b, t, d, None if q_weight is None else q_weight.data_ptr(),
          None if k_weight is None else k_weight.data_ptr(), eps, positions.data_ptr(), positions.dtype is torch.int64,
          plan._ptr, plan.magnitude, plan.rot_dim, plan.interleaved)
    return q_out, k_out


# ---------------------------------------------------------------- the cache
class KVCacheInt8:
    """A paged int8 KV cache: ``k``, ``v`` int8 [layers?, pages, heads, page, D] and ``k_scale``, ``v_scale``
    fp32 [layers?, pages, heads, page], contiguous on one CUDA device.  ``layer(i)`` is one layer's view."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "layers", "pages", "heads", "page", "head_dim", "device", "_ptrs",
                 "_dims")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        if not all(x.is_cuda for x in (k, v, k_scale, v_scale)):
            raise RuntimeError("the cache must be CUDA")
        if k.dtype != torch.int8 or v.dtype != torch.int8:
            raise RuntimeError("cache codes must be int8")
        if k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32:
            raise RuntimeError("cache scales must be fp32")
        if k.dim() not in (4, 5):
            raise RuntimeError("cache codes must be [layers?, pages, heads, page, D]")
        if v.shape != k.shape or k_scale.shape != k.shape[:-1] or v_scale.shape != k.shape[:-1]:
            raise RuntimeError("cache tensors must have the same layers, pages, heads and page size")
        if not all(x.is_contiguous() for x in (k, v, k_scale, v_scale)):
            raise RuntimeError("cache tensors must be contiguous")
        if any(x.device != k.device for x in (v, k_scale, v_scale)):
            raise RuntimeError("cache tensors must be on one device")
        if not 1 <= k.shape[-1] <= MAX_HEAD_DIM:
            raise RuntimeError(f"the cache's head dimension must be 1 to {MAX_HEAD_DIM}")
        if k.shape[-2] < 1 or k.shape[-3] < 1:
            raise RuntimeError("the cache's page and head counts must be positive")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.layers = k.shape[0] if k.dim() == 5 else None
        self.pages, self.heads, self.page, self.head_dim = k.shape[-4:]
        self.device = k.device
        self._ptrs = (k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr())
        self._dims = (self.pages, self.heads, self.page, self.head_dim)

    @classmethod
    def empty(cls, pages: int, heads: int, page: int, head_dim: int, layers: int | None = None,
              device="cuda") -> "KVCacheInt8":
        """A cache of zeros."""
        shape = (pages, heads, page, head_dim) if layers is None else (layers, pages, heads, page, head_dim)
        return cls(torch.zeros(shape, dtype=torch.int8, device=device),
                   torch.zeros(shape, dtype=torch.int8, device=device),
                   torch.zeros(shape[:-1], dtype=torch.float32, device=device),
                   torch.zeros(shape[:-1], dtype=torch.float32, device=device))

    def layer(self, i: int) -> "KVCacheInt8":
        if self.layers is None:
            raise RuntimeError("the cache has no layers")
        return KVCacheInt8(self.k[i], self.v[i], self.k_scale[i], self.v_scale[i])

    def _one_layer(self, op: str) -> None:
        if self.layers is not None:
            raise RuntimeError(f"{op}: takes one layer of the cache; pass cache.layer(i)")


def _ints(x: torch.Tensor, name: str, shape: tuple, dev: torch.device) -> torch.Tensor:
    """A contiguous int32 tensor of that shape."""
    if x is None:
        raise RuntimeError(f"{name} must be {list(shape)}")
    if x.dtype is not torch.int32 or x.device != dev:
        raise RuntimeError(f"{name} must be int32 on the cache's device")
    if x.shape != shape:
        raise RuntimeError(f"{name} must be {list(shape)}")
    return x if x.is_contiguous() else x.contiguous()


def _table(table: torch.Tensor, dev: torch.device) -> tuple[torch.Tensor, int, int, int]:
    """(table, its sequences, row stride, columns)"""
    if table.dtype is not torch.int32 or table.device != dev:
        raise RuntimeError("table must be int32 on the cache's device")
    if table.dim() != 2:
        raise RuntimeError("table must be [B, pages of a sequence]")
    b, cols = table.shape
    ld, unit = table.stride()
    if unit != 1 or ld < cols:
        table = table.contiguous()
        ld = cols
    return table, b, ld, cols


def _write(q, k, v, positions, plan, cache, table, start, counts, op):
    if cache.layers is not None:
        cache._one_layer(op)
    dev = cache.device
    if k.dim() != 4:
        raise RuntimeError(f"{op}: k must be [B, T, heads, D]")
    lead = k.shape[:2]
    k, kshape, b, t, kb, kt, kh = _rows(k, "k", lead)
    v, vshape, _, _, vb, vt, vh = _rows(v, "v", lead)
    d, dt = cache.head_dim, k.dtype
    if kshape[2] != cache.heads or kshape[3] != d or vshape != kshape:
        raise RuntimeError(f"{op}: k and v must be [B, T, {cache.heads}, {d}] like the cache")
    if v.dtype is not dt or k.device != dev or v.device != dev:
        raise RuntimeError(f"{op}: k and v must share one dtype and be on the cache's device")
    table, rows, ld, cols = _table(table, dev)
    if rows != b:
        raise RuntimeError(f"{op}: table must have a row for each of {b} sequences")
    start = _ints(start, "start", (b,), dev)
    if counts is not None:
        counts = _ints(counts, "counts", (b,), dev)
    q_out, qp, qb, qt, qh, hq, qop = None, None, 0, 0, 0, 0, None
    pp, p64, sp, mag, rot, inter = None, 0, None, 1.0, 0, 0
    if plan is not None:
        q, qshape, _, _, qb, qt, qh = _rows(q, "q", lead)
        if q.dtype is not dt or q.device != dev or qshape[3] != d:
            raise RuntimeError(f"{op}: q must have k's dtype, device and head dimension")
        if plan.device != dev or plan.rot_dim > d:
            raise RuntimeError(f"{op}: the plan must be on the cache's device with rot_dim <= D")
        positions = _positions(positions, lead, dev)
        hq = qshape[2]
        q_out = _new(qshape, dt, dev)
        qp, qop = q.data_ptr(), q_out.data_ptr()
        pp, p64, sp = positions.data_ptr(), positions.dtype is torch.int64, plan._ptr
        mag, rot, inter = plan.magnitude, plan.rot_dim, plan.interleaved
    _call(op, dev, lib.bw_rotary_kv_write_int8, qp, qb, qt, qh, hq, k.data_ptr(), kb, kt, kh, v.data_ptr(), vb, vt, vh,
          qop, DTYPE_CODE[dt], b, t, pp, p64, sp, mag, rot, inter, *cache._ptrs, *cache._dims, table.data_ptr(), ld, cols,
          start.data_ptr(), None if counts is None else counts.data_ptr())
    return q_out


def kv_write_int8(k: torch.Tensor, v: torch.Tensor, cache: KVCacheInt8, table: torch.Tensor, start: torch.Tensor,
                  counts: torch.Tensor | None = None) -> None:
    """Quantise k, v [B, T, heads, D] (fp16 or bf16) into the cache: token i of sequence b goes to slot
    ``start[b] + i`` (``i < counts[b]`` where counts are given).  One fp32 scale per token and head,
    ``max|x| / 127``; codes ``clamp(rne(x / scale), -127, 127)``; NaN is ignored by the scale and coded 0."""
    _write(None, k, v, None, None, cache, table, start, counts, "kv_write_int8")


def rotary_kv_write_int8(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, plan: RotaryPlan,
                         cache: KVCacheInt8, table: torch.Tensor, start: torch.Tensor,
                         counts: torch.Tensor | None = None) -> torch.Tensor:
    """``rotary`` of q [B, T, Hq, D] and k, and ``kv_write_int8`` of the rotated k and v, in one launch.

    The rotated keys are quantised from their 32-bit values.  Returns the rotated q (every token's,
    ``counts`` limits the write only)."""
    return _write(q, k, v, positions, plan, cache, table, start, counts, "rotary_kv_write_int8")


def norm_rotary_kv_write_int8(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                              plan: RotaryPlan, cache: KVCacheInt8, table: torch.Tensor, start: torch.Tensor,
                              q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                              eps: float = 1e-6, counts: torch.Tensor | None = None,
                              offsets: torch.Tensor | None = None,
                              keys: bool = False) -> tuple[torch.Tensor, torch.Tensor | None]:
    """``norm_rotary`` of q and k, and ``kv_write_int8`` of the normalised and rotated k and of v, in one launch.

    q [B, T, Hq, D] with k, v [B, T, heads, D] as in ``rotary_kv_write_int8``; or, with ``offsets`` [B + 1] (int32, not
    descending), packed prompts [N, .., D]: rows ``offsets[b] .. offsets[b + 1]`` are sequence b's and go to slots
    ``start[b]`` on, other rows are not written.  The keys are quantised from their 32-bit values.  Returns the rotated q and,
    with ``keys``, the rotated k (every row's), else None."""
    op = "norm_rotary_kv_write_int8"
    if cache.layers is not None:
        cache._one_layer(op)
    dev = cache.device
    packed = offsets is not None
    if k.dim() != (3 if packed else 4):
        raise RuntimeError(f"{op}: k must be {'[N, heads, D] with offsets' if packed else '[B, T, heads, D]'}")
    lead = k.shape[:-2]
    q, qshape, _, _, qb, qt, qh = _rows(q, "q", lead)
    k, kshape, b, t, kb, kt, kh = _rows(k, "k", lead)
    v, vshape, _, _, vb, vt, vh = _rows(v, "v", lead)
    d, dt = cache.head_dim, k.dtype
    if kshape[-2] != cache.heads or kshape[-1] != d or vshape != kshape:
        raise RuntimeError(f"{op}: k and v must be [.., {cache.heads}, {d}] like the cache")
    if v.dtype is not dt or k.device != dev or v.device != dev:
        raise RuntimeError(f"{op}: k and v must share one dtype and be on the cache's device")
    if q.dtype is not dt or q.device != dev or qshape[-1] != d:
        raise RuntimeError(f"{op}: q must have k's dtype, device and head dimension")
    if plan.device != dev or plan.rot_dim > d:
        raise RuntimeError(f"{op}: the plan must be on the cache's device with rot_dim <= D")
    if not eps >= 0:
        raise RuntimeError(f"{op}: eps must not be negative")
    table, rows, ld, cols = _table(table, dev)
    if packed:
        if counts is not None:
            raise RuntimeError(f"{op}: packed rows have offsets, no counts")
        b = rows
        offsets = _ints(offsets, "offsets", (b + 1,), dev)
    elif rows != b:
        raise RuntimeError(f"{op}: table must have a row for each of {b} sequences")
    start = _ints(start, "start", (b,), dev)
    if counts is not None:
        counts = _ints(counts, "counts", (b,), dev)
    positions = _positions(positions, lead, dev)
    q_weight, k_weight = _weight(q_weight, "q_weight", d, dt, dev), _weight(k_weight, "k_weight", d, dt, dev)
    q_out = _new(qshape, dt, dev)
    k_out = _new(kshape, dt, dev) if keys else None
    _call(op, dev, lib.bw_norm_rotary_kv_write_int8, q.data_ptr(), qb, qt, qh, qshape[-2], k.data_ptr(), kb, kt, kh,
          v.data_ptr(), vb, vt, vh, q_out.data_ptr(), k_out.data_ptr() if keys else None, DTYPE_CODE[dt], b, t,
          None if q_weight is None else q_weight.data_ptr(), None if k_weight is None else k_weight.data_ptr(), eps,
          positions.data_ptr(), positions.dtype is torch.int64, plan._ptr, plan.magnitude, plan.rot_dim, plan.interleaved,
          *cache._ptrs, *cache._dims, table.data_ptr(), ld, cols, start.data_ptr(),
          None if counts is None else counts.data_ptr(), offsets.data_ptr() if packed else None)
    return q_out, k_out


def kv_read_int8(cache: KVCacheInt8, table: torch.Tensor, start: torch.Tensor | None, n: int,
                 lens: torch.Tensor | None = None, dtype: torch.dtype = torch.float16) -> tuple[torch.Tensor, torch.Tensor]:
    """Values of slots ``start[b] + i``, i < n (start None: 0): k, v [layers?, B, n, heads, D] in ``dtype``.
    Slots ``i >= lens[b]`` are zeros where ``lens`` are given."""
    dev = cache.device
    if dtype not in _HALF:
        raise RuntimeError("kv_read_int8: dtype must be fp16 or bf16")
    if n < 0:
        raise RuntimeError("kv_read_int8: n must not be negative")
    table, b, ld, cols = _table(table, dev)
    sp = None if start is None else _ints(start, "start", (b,), dev)
    lp = None if lens is None else _ints(lens, "lens", (b,), dev)
    layers = cache.layers
    shape = (b, n, cache.heads, cache.head_dim) if layers is None else (layers, b, n, cache.heads, cache.head_dim)
    k, v = _new(shape, dtype, dev), _new(shape, dtype, dev)
    _call("kv_read_int8", dev, lib.bw_kv_read_int8, *cache._ptrs, 1 if layers is None else layers, *cache._dims,
          table.data_ptr(), ld, cols, None if sp is None else sp.data_ptr(), None if lp is None else lp.data_ptr(), b, n,
          k.data_ptr(), v.data_ptr(), DTYPE_CODE[dtype])
    return k, v


def kv_move_int8(cache: KVCacheInt8, table: torch.Tensor, start: torch.Tensor, path: torch.Tensor,
                 taken: torch.Tensor) -> None:
    """Move the accepted nodes of draft trees to their final slots, in every layer of the cache.

    The tree of sequence b lies at slots ``start[b] + node``; nodes ``path[b, :taken[b]]`` (as
    ``verify_tree`` gives them) go to slots ``start[b] + 1, start[b] + 2, ..``."""
    dev = cache.device
    table, b, ld, cols = _table(table, dev)
    if path.dim() != 2 or path.shape[1] > MAX_NODES:
        raise RuntimeError(f"path must be [B, T] with T <= {MAX_NODES}")
    t = path.shape[1]
    path = _ints(path, "path", (b, t), dev)
    start, taken = _ints(start, "start", (b,), dev), _ints(taken, "taken", (b,), dev)
    _call("kv_move_int8", dev, lib.bw_kv_move_int8, *cache._ptrs, 1 if cache.layers is None else cache.layers,
          *cache._dims, table.data_ptr(), ld, cols, start.data_ptr(), path.data_ptr(), t, taken.data_ptr(), b, t)


# ---------------------------------------------------------------- trees
def tree_positions(parents: torch.Tensor, ctx_lens: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Masks [B, T] int64 and positions [B, T] int32 of draft trees.

    ``parents`` [B, T] int32, T <= 64: node 0 is the root, ``parents[b, i] < i`` is node i's parent;
    any other value takes the node out of the tree (mask 0).  Bit j of a mask: node j is the node
    itself or an ancestor.  Positions are ``ctx_lens[b]`` (0 without) plus the node's depth."""
    if not parents.is_cuda or parents.dtype != torch.int32:
        raise RuntimeError("parents must be CUDA int32")
    if parents.dim() != 2 or parents.shape[1] > MAX_NODES:
        raise RuntimeError(f"parents must be [B, T] with T <= {MAX_NODES}")
    dev = parents.device
    parents = parents.contiguous()
    b, t = parents.shape
    if ctx_lens is not None:
        ctx_lens = _ints(ctx_lens, "ctx_lens", (b,), dev)
    mask, pos = _new((b, t), torch.int64, dev), _new((b, t), torch.int32, dev)
    _call("tree_positions", dev, lib.bw_tree_positions, parents.data_ptr(), t,
          None if ctx_lens is None else ctx_lens.data_ptr(), b, t, mask.data_ptr(), pos.data_ptr())
    return mask, pos


def tree_attention_int8(q: torch.Tensor, cache: KVCacheInt8, table: torch.Tensor, ctx_lens: torch.Tensor,
                        mask: torch.Tensor | None = None, counts: torch.Tensor | None = None,
                        softmax_scale: float | None = None) -> torch.Tensor:
    """Attention of the nodes of draft trees over the cache: q [B, T, Hq, D] -> [B, T, Hq, D].

    Node i of sequence b sees the slots before ``ctx_lens[b]`` and the slots ``ctx_lens[b] + j`` of the
    nodes j whose bit is set in ``mask[b, i]`` (int64; None: nodes 0 .. i, a chain).  ``counts`` [B]
    limits a sequence's nodes: later ones are not seen and give zeros, and so does a node that sees
    nothing.  Query head h reads key head ``h // (Hq / heads)``.  T <= 64; T = 1 is ordinary decoding.
    ``softmax_scale`` defaults to ``D ** -0.5``.

    The tensor-core kernel takes D = 64 or 128, pages of 16, 32, 64 or a multiple of 128 slots, cache tensors on
    16-byte boundaries with fewer than 2^31 rows (pages * heads * page), and at most 32768 query rows a key head; other
    calls go to a kernel of a CTA a query row, some 25 times slower on long batches."""
    if cache.layers is not None:
        cache._one_layer("tree_attention_int8")
    dev, dt = cache.device, q.dtype
    if not q.is_cuda or dt not in _HALF:
        raise RuntimeError("q must be CUDA fp16 or bf16")
    if q.dim() != 4 or q.device != dev:
        raise RuntimeError("q must be [B, T, heads, D] on the cache's device")
    shape = q.shape
    b, t, hq, d = shape
    heads = cache.heads
    if d != cache.head_dim:
        raise RuntimeError(f"q must have the cache's head dimension {cache.head_dim}")
    if hq == 0 or hq % heads:
        raise RuntimeError(f"q's heads must be a multiple of the cache's {heads}")
    if t > MAX_NODES:
        raise RuntimeError(f"at most {MAX_NODES} nodes a sequence")
    stride = q.stride()
    if stride[3] != 1 and d > 1:
        q = q.contiguous()
        stride = q.stride()
    table, rows, ld, cols = _table(table, dev)
    if rows != b:
        raise RuntimeError(f"table must have a row for each of {b} sequences")
    ctx_lens = _ints(ctx_lens, "ctx_lens", (b,), dev)
    if counts is not None:
        counts = _ints(counts, "counts", (b,), dev)
    if mask is not None:
        if mask.dtype is not torch.int64 or mask.device != dev or mask.shape != (b, t):
            raise RuntimeError(f"mask must be int64 [{b}, {t}] on the cache's device")
        if not mask.is_contiguous():
            mask = mask.contiguous()
    out = _new(shape, dt, dev)
    if b == 0 or t == 0:
        return out
    nbytes = _attention_bytes(dev.index, b, t, hq, heads, d)
    ws = _workspace(dev, nbytes) if nbytes else None
    _call("tree_attention_int8", dev, lib.bw_tree_attention_int8, q.data_ptr(), stride[0], stride[1], stride[2],
          DTYPE_CODE[dt], out.data_ptr(), *cache._ptrs, *cache._dims, table.data_ptr(), ld, cols, ctx_lens.data_ptr(),
          None if mask is None else mask.data_ptr(), None if counts is None else counts.data_ptr(), b, t, hq,
          d ** -0.5 if softmax_scale is None else float(softmax_scale), None if ws is None else ws.data_ptr(),
          0 if ws is None else nbytes)
    return out


def verify_tree(target_probs: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor, accept_u: torch.Tensor,
                sample_e: torch.Tensor, draft_probs: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Accept drafted tokens so that what comes out is distributed as the target alone would draw it.

    ``target_probs`` [B, T, V] fp32: row i is the target's distribution of the token after node i;
    ``tokens`` [B, T] int64 and ``parents`` [B, T] int32: the tree, node 0 (the root) the last
    committed token; ``draft_probs`` [B, T, V] fp32: row i is the distribution from which node i's
    children were drawn (None: drafts without one, as from a lookup); ``accept_u`` [B, T] uniform on
    [0, 1), ``sample_e`` [B, V] exponential.

    From the root, with w = target and Z = 1, a node's children are tried in index order: child i
    with token x is taken if ``u_i * draft(x) * Z < w(x)``, else ``w = max(w - Z * draft, 0)`` (without
    drafts' distribution draft(x) = 1 and w(x) = 0) and ``Z = sum(w)``.  Where no child is taken the
    last token is ``argmax(w / e)``, ties to the lowest.  Z is summed in one order for every B, so a
    sequence's tokens do not depend on its batch.

    Returns ``n`` [B] int32 accepted nodes, ``path`` [B, T] int32 (the nodes, then -1) and ``out`` [B, T]
    int64 (their tokens, the last token, then -1)."""
    dev = target_probs.device
    if not target_probs.is_cuda or target_probs.dtype != torch.float32:
        raise RuntimeError("target_probs must be CUDA fp32")
    if target_probs.dim() != 3 or target_probs.shape[2] == 0:
        raise RuntimeError("target_probs must be [B, T, V]")
    b, t, v = target_probs.shape
    if t > MAX_NODES:
        raise RuntimeError(f"at most {MAX_NODES} nodes a sequence")
    nodes, row = (b, t), (b, v)
    if tokens.dtype is not torch.int64 or tokens.device != dev or tokens.shape != nodes:
        raise RuntimeError(f"tokens must be int64 [{b}, {t}] on the probabilities' device")
    if parents.dtype is not torch.int32 or parents.device != dev or parents.shape != nodes:
        raise RuntimeError(f"parents must be int32 [{b}, {t}] on the probabilities' device")
    if accept_u.dtype is not torch.float32 or accept_u.device != dev or accept_u.shape != nodes:
        raise RuntimeError(f"accept_u must be fp32 [{b}, {t}] on the probabilities' device")
    if sample_e.dtype is not torch.float32 or sample_e.device != dev or sample_e.shape != row:
        raise RuntimeError(f"sample_e must be fp32 [{b}, {v}] on the probabilities' device")
    if draft_probs is not None:
        if draft_probs.dtype != torch.float32 or draft_probs.device != dev or draft_probs.shape != target_probs.shape:
            raise RuntimeError("draft_probs must be fp32 of target_probs' shape and device")
        draft_probs = draft_probs.contiguous()
    target_probs, tokens, parents = target_probs.contiguous(), tokens.contiguous(), parents.contiguous()
    accept_u, sample_e = accept_u.contiguous(), sample_e.contiguous()
    n, path, out = _new((b,), torch.int32, dev), _new(nodes, torch.int32, dev), _new(nodes, torch.int64, dev)
    if b and not t:
        n.zero_()
    _call("verify_tree", dev, lib.bw_verify_tree, target_probs.data_ptr(),
          None if draft_probs is None else draft_probs.data_ptr(), tokens.data_ptr(),
          parents.data_ptr(), accept_u.data_ptr(), sample_e.data_ptr(), b, t, v, n.data_ptr(), path.data_ptr(),
          out.data_ptr())
    return n, path, out


__all__ = ["MAX_NODES", "KVCacheInt8", "RotaryPlan", "kv_move_int8", "kv_read_int8", "kv_write_int8", "norm_rotary",
           "norm_rotary_kv_write_int8", "reset_workspaces",
           "rotary", "rotary_frequencies", "rotary_kv_write_int8", "rotary_plan", "tree_attention_int8",
           "tree_positions", "verify_tree"]
