"""Scratch memory of the operators whose kernels count on words that are zero before a call and zero after it.

Outside stream captures there is one tensor per (device, stream), replaced by a larger one when a call needs more: the
calls of a stream follow one another, and the allocator gives a freed block to later work of the same stream only.

A CUDA graph keeps the addresses of its capture for as long as it lives, may be replayed on any stream, and runs
nothing of what came before its capture.  So a capture never gets that tensor.  Each capture has its own, one per
stream that it captures: it lies in the graph's memory pool, and its words are cleared by the graph itself at the
start of each replay.
"""
from __future__ import annotations

import ctypes
import threading

import torch

from ._lib import check, lib

_LEAST = 1 << 20


def capture_id(index: int, stream: int) -> int:
    """0, or the id of the capture that ``stream``, the current stream of device ``index``, is part of."""
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            return capture_id(index, stream)
    if not torch.cuda.is_current_stream_capturing():
        return 0
    found = ctypes.c_uint64(0)
    check(lib.bw_stream_capture_id(stream, ctypes.byref(found)), "stream_capture_id")
    return found.value


class Workspaces:
    """``zeroed``: how many bytes of a workspace a kernel counts on, from its beginning (None: all)."""

    def __init__(self, zeroed: int | None = None):
        self._zeroed = zeroed
        self._lock = threading.Lock()
        self.eager: dict[tuple[int, int], torch.Tensor] = {}
        self._captured: dict[tuple[int, int], tuple[int, torch.Tensor]] = {}

    def get(self, dev: torch.device, stream: int, nbytes: int) -> torch.Tensor:
        """At least ``nbytes`` for one call on ``stream``, the current stream of ``dev``."""
        index = dev.index if dev.index is not None else torch.cuda.current_device()
        key = (index, stream)
        capture = capture_id(index, stream)
        if not capture:
            ws = self.eager.get(key)
            if ws is None or ws.numel() < nbytes:
                with self._lock:
                    ws = self.eager[key] = torch.zeros(max(nbytes, _LEAST), dtype=torch.uint8, device=dev)
            return ws
        with self._lock:
            last, ws = self._captured.get(key, (0, None))
            if last != capture or ws.numel() < nbytes:
                ws = torch.empty(max(nbytes, _LEAST), dtype=torch.uint8, device=dev)
                ws[:self._zeroed].zero_()
                self._captured[key] = capture, ws
        return ws

    def reset(self) -> None:
        """Zero every workspace outside graphs (a graph clears its own)."""
        with self._lock:
            for ws in self.eager.values():
                ws.zero_()
