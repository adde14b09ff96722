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
from .mla_q4 import _keep_plan, _layout, _per_sequence, _plans

MAX_BUFFERS = 8


def cache_evict(weight: torch.Tensor, buffers, keep: int, lengths: torch.Tensor | int | None = None, sink: int = 0,
                recent: int = 0, capacity: int | None = None):
    """-> (new buffers [B, capacity, ...], index [B, keep] int32, lengths [B] int32).

    weight fp32 [B, cap]; buffers: up to 8 tensors [B, cap, ...] on the same device.  ``lengths``: the sequences' lengths, a
    whole number for all or an int32 [B] device tensor (default: cap).  min(length, keep) positions stay (sink + recent
    <= keep): ties go to the lowest position, a NaN weight counts below all others.  index: the positions that stayed, ascending, then -1.
    Rows past a sequence's new length are zero.  ``capacity``: rows of the new buffers (default: keep).
    """
    buffers = list(buffers)
    length = lengths if not isinstance(lengths, torch.Tensor) else None
    if length is not None:
        lengths = None
    key = (weight.shape, weight.stride(), weight.dtype, keep, length, _layout(lengths), sink, recent, capacity,
           *[(x.shape, x.stride(), x.dtype) for x in buffers])
    (B, cap, keep, sink, recent, rows, most, w_pitch, direct, shapes, arrays, ptrs) = _plans.get(key) or _keep_plan(
        key, _evict_plan(weight, buffers, keep, length, lengths, sink, recent, capacity))
    T.require_device(weight, lengths, *buffers)
    if T.tracked(*buffers):
        raise ValueError("cache_evict carries no gradient: call it under no_grad or on detached buffers")
    if w_pitch is None:
        weight, w_pitch = weight.contiguous(), cap
    if not all(direct):
        # (their layout is the key's: a copy's pitches are those of a contiguous buffer, which the plan holds)
        buffers = [x if ok else x.contiguous() for x, ok in zip(buffers, direct)]
    new = [x.new_empty(s) for x, s in zip(buffers, shapes)]
    index, kept = weight.new_empty((B, keep), dtype=torch.int32), weight.new_empty(B, dtype=torch.int32)
    if B == 0:
        return new, index, kept
    src_b, src_r, dst_b, dst_r, size = arrays
    with T.current(weight.device):
        _lib.call("k3_cache_evict", weight.data_ptr(), w_pitch, T.ptr(lengths), most, B, keep, sink, recent, index.data_ptr(),
                  kept.data_ptr(), len(new), ptrs(*[x.data_ptr() for x in buffers]), src_b, src_r, ptrs(*[x.data_ptr() for x in new]),
                  dst_b, dst_r, size, rows, T.stream(weight))
    return new, index, kept


def _evict_plan(weight, buffers, keep, length, lengths, sink, recent, capacity) -> tuple:
    if weight.dim() != 2:
        raise ValueError(f"weight must be [B, cap]; got {tuple(weight.shape)}")
    if weight.dtype != torch.float32:
        raise TypeError(f"weight must be float32; got {weight.dtype}")
    B, cap = weight.shape
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
    most = cap
    if length is not None:
        most = int(length)
        if not 0 <= most <= cap:
            raise ValueError(f"length {most} outside the capacity {cap}")
    _per_sequence(lengths, B, "lengths")
    width = [math.prod(x.shape[2:]) for x in buffers]
    size = [n * x.element_size() for n, x in zip(width, buffers)]
    direct, src_b, src_r = [], [], []
    for x, n in zip(buffers, width):
        ok = B == 0 or cap == 0 or (x[0, 0].is_contiguous() and (cap < 2 or x.stride(1) >= n) and (B < 2 or x.stride(0) >= 0))
        e = x.element_size()
        direct.append(ok)
        src_b.append((x.stride(0) if ok else cap * n) * e if B > 1 else 0)
        src_r.append((x.stride(1) if ok else n) * e if cap > 1 else n * e)
    longs = ctypes.c_int64 * max(len(buffers), 1)
    return (B, cap, keep, sink, recent, rows, most, None if cap > 1 and weight.stride(1) != 1 else weight.stride(0) if B > 1 else 0,
            tuple(direct), tuple((B, rows, *x.shape[2:]) for x in buffers),
            (longs(*src_b), longs(*src_r), longs(*[rows * s for s in size]), longs(*size), longs(*size)),
            ctypes.c_void_p * max(len(buffers), 1))
