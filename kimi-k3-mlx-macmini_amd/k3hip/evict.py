"""Eviction from a cache by accumulated attention weight.

``cache_evict(weight, buffers, keep, ...)`` keeps, of every sequence, the first ``sink`` positions, the last ``recent`` and
those of the rest that received the most attention (``weight``, as ``k3hip.mla_q4.mla_q4_attention`` sums it), and moves
their rows to the front of new buffers in their order.  It works on any buffers [B, cap, ...] with contiguous rows: the 4-bit
cache's, the bf16 or fp32 cache's (``MLACache.latent``, ``.rot``), the weights themselves.  The reference's cache only grows
(``air_llm/models/kimi_k3/attention_mla.py:62-117``).
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from . import _torch as T
from .mla_q4 import _per_sequence

MAX_BUFFERS = 8


def cache_evict(weight: torch.Tensor, buffers, keep: int, lengths: torch.Tensor | int | None = None, sink: int = 0,
                recent: int = 0, capacity: int | None = None):
    """-> (new buffers [B, capacity, ...], index [B, keep] int32, lengths [B] int32).

    weight fp32 [B, cap]; buffers: up to 8 tensors [B, cap, ...] on the same device.  ``lengths``: the sequences' lengths, a
    whole number for all or an int32 [B] device tensor (default: cap).  min(length, keep) positions stay (sink + recent
    <= keep): ties go to the lowest position, a NaN weight counts below all others.  index: the positions that stayed, ascending, then -1.
    Rows past a sequence's new length are zero.  ``capacity``: rows of the new buffers (default: keep).
    """
    if weight.dim() != 2:
        raise ValueError(f"weight must be [B, cap]; got {tuple(weight.shape)}")
    if weight.dtype != torch.float32:
        raise TypeError(f"weight must be float32; got {weight.dtype}")
    B, cap = weight.shape
    buffers = list(buffers)
    if len(buffers) > MAX_BUFFERS:
        raise ValueError(f"at most {MAX_BUFFERS} buffers; got {len(buffers)}")
    keep, sink, recent = int(keep), int(sink), int(recent)
    if keep < 0 or sink < 0 or recent < 0 or sink + recent > keep:
        raise ValueError(f"keep={keep} must hold sink={sink} and recent={recent}, none of them negative")
    rows = keep if capacity is None else int(capacity)
    if rows < keep:
        raise ValueError(f"capacity {rows} < keep {keep}")
    for x in buffers:
        if x.dim() < 2 or tuple(x.shape[:2]) != (B, cap):
            raise ValueError(f"buffers must be [{B}, {cap}, ...]; got {tuple(x.shape)}")
        if x.requires_grad and torch.is_grad_enabled():
            raise ValueError("cache_evict carries no gradient: call it under no_grad or on detached buffers")
    T.require_device(weight, *buffers)
    device, most = weight.device, cap
    if lengths is not None and not isinstance(lengths, torch.Tensor):
        most, lengths = int(lengths), None
        if not 0 <= most <= cap:
            raise ValueError(f"length {most} outside the capacity {cap}")
    lengths = _per_sequence(lengths, B, "lengths", device)
    if cap > 1 and weight.stride(1) != 1:
        weight = weight.contiguous()
    src = [x if x[0, :1].is_contiguous() and (cap < 2 or x.stride(1) >= math.prod(x.shape[2:])) else x.contiguous()
           for x in buffers] if B else buffers
    new = [torch.empty((B, rows, *x.shape[2:]), dtype=x.dtype, device=device) for x in buffers]
    index = torch.empty((B, keep), dtype=torch.int32, device=device)
    kept = torch.empty(B, dtype=torch.int32, device=device)
    if B == 0:
        return new, index, kept
    n = len(src)
    size = [math.prod(x.shape[2:]) * x.element_size() for x in src]
    longs, ptrs = ctypes.c_int64 * max(n, 1), ctypes.c_void_p * max(n, 1)
    src_b = longs(*[x.stride(0) * x.element_size() if B > 1 else 0 for x in src])
    src_r = longs(*[x.stride(1) * x.element_size() if cap > 1 else s for x, s in zip(src, size)])
    dst_b, dst_r = longs(*[rows * s for s in size]), longs(*size)
    with T.current(device):
        _lib.call("k3_cache_evict", T.ptr(weight), weight.stride(0) if B > 1 else 0, T.ptr(lengths), most, B, keep, sink, recent,
                  T.ptr(index), T.ptr(kept), n, ptrs(*[x.data_ptr() for x in src]), src_b, src_r,
                  ptrs(*[x.data_ptr() for x in new]), dst_b, dst_r, longs(*size), rows, T.stream(weight))
    return new, index, kept
