"""The 4-bit latent cache: writing it and attending over it.

A cached position holds its 512 latent values as MXFP4 -- ``packed`` [256] u8 E2M1 codes and
``scales`` [16] u8 E8M0 bytes, the format of ``k3hip.mxfp4`` -- and its 64 rotary values in bf16:
400 bytes where the bf16 cache takes 1152.  The counterpart of the reference's optional quantised
latent (``air_llm/models/kimi_k3/mla_quant.py:64-116``; group-affine there), which keeps the rotary
part unquantised as well.

``mla_q4_append`` rounds new latents into a batch of such caches, ``mla_q4_attention`` is the absorbed
latent attention of one token or several of each sequence over them (``attention_mla.py:193-212``),
and sums, if asked to, the attention weight that every position received, by which
``k3hip.evict.cache_evict`` chooses what stays.  ``MLACacheQ4`` holds such a cache as ``k3hip.mla.MLACache`` does the bf16
one; ``k3hip.mla.MLAAttention`` runs on either.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib, _workspace
from . import _torch as T

LATENT, ROPE, GROUP = 512, 64, 32
# Scratch up to this size is kept per stream (a decode step's); larger scratch, a prompt's, is the call's own, and so is a captured call's.
KEPT_WORKSPACE = 1 << 26
MAX_ROWS, MAX_SEQUENCES = 1 << 16, (1 << 16) - 1      # heads x sequences, and sequences, of one k3_mla_q4_attention


# What a call's layout (shapes, strides, dtypes; no addresses) comes to, once its checks are passed: the checks cost
# more than a short call's kernels.
_plans: dict[tuple, tuple] = {}
MAX_PLANS = 4096


def _keep_plan(key: tuple, plan: tuple) -> tuple:
    if len(_plans) >= MAX_PLANS:
        _plans.clear()
    _plans[key] = plan
    return plan


def _buffers(packed, scales, rot):
    """The cache's three buffers as [B, cap, .]: dtypes, shapes and row layout."""
    for t, name, width, dtype in ((packed, "packed", LATENT // 2, torch.uint8), (scales, "scales", LATENT // GROUP, torch.uint8),
                                  (rot, "rot", ROPE, torch.bfloat16)):
        if t.dtype != dtype:
            raise TypeError(f"{name} must be {dtype}; got {t.dtype}")
        if t.dim() != 3 or t.shape[2] != width:
            raise ValueError(f"{name} must be [B, cap, {width}]; got {tuple(t.shape)}")
        if t.shape[1] and t.stride(2) != 1:
            raise ValueError(f"{name}: the values of a position must be contiguous")
    if packed.shape[:2] != scales.shape[:2] or packed.shape[:2] != rot.shape[:2]:
        raise ValueError(f"packed {tuple(packed.shape)}, scales {tuple(scales.shape)} and rot {tuple(rot.shape)} differ in batch "
                         "or capacity")
    return packed.shape[:2]


def _per_sequence(v: torch.Tensor | None, B: int, name: str) -> None:
    """Refuses what is neither None nor a contiguous int32 [B] tensor."""
    if v is None:
        return
    if v.dtype != torch.int32:
        raise TypeError(f"{name} must be an int32 tensor; got {v.dtype}")
    if tuple(v.shape) != (B,) or not v.is_contiguous():
        raise ValueError(f"{name} must be a contiguous [{B}]; got {tuple(v.shape)}")


def _layout(t: torch.Tensor | None):
    return None if t is None else (t.shape, t.stride(), t.dtype)


def _pitches(t: torch.Tensor) -> tuple[int, int]:
    """Batch and row pitch in elements; a pitch that is never used may be anything."""
    return (t.stride(0) if t.shape[0] > 1 else 0), (t.stride(1) if t.shape[1] > 1 else max(t.stride(1), t.shape[2]))


def _apart(t: torch.Tensor, name: str) -> None:
    """Refuses a buffer [B, cap, ...] to be written whose sequences share memory (an expanded one): they would race."""
    B, cap = t.shape[:2]
    if B < 2 or cap == 0:
        return
    batch, row, width = t.stride(0), t.stride(1), t.shape[2] if t.dim() == 3 else 1
    if batch < (cap - 1) * row + width and (batch < width or (cap > 1 and row < (B - 1) * batch + width)):
        raise ValueError(f"{name}: the sequences overlap in memory (strides {t.stride()}); they are written")


def _weight_pitch(weight: torch.Tensor | None, B: int, cap: int) -> int:
    """The batch pitch of the accumulated attention, [B, cap] fp32 or None."""
    if weight is None:
        return 0
    if weight.dtype != torch.float32:
        raise TypeError(f"weight must be float32; got {weight.dtype}")
    if tuple(weight.shape) != (B, cap) or (cap > 1 and weight.stride(1) != 1):
        raise ValueError(f"weight must be [{B}, {cap}] with contiguous rows; got {tuple(weight.shape)}")
    _apart(weight, "weight")
    return weight.stride(0) if B > 1 else 0


def scratch(device: torch.device, nbytes: int, tag: str) -> torch.Tensor:
    """Workspace of a call on device, the current one.  A captured call's is its graph's, also where the stream has a kept one: two graphs
    captured after a call there may replay side by side, and one would take the other's list of ranges."""
    if nbytes > KEPT_WORKSPACE or T.capturing():
        return torch.empty(nbytes, dtype=torch.uint8, device=device)
    return _workspace.get(device, nbytes, tag)


def _rows_ok(t: torch.Tensor, per: int) -> bool:
    """Contiguous rows, pitches of whole 16 bytes (``per`` elements): read as they are where the base is aligned too."""
    return t.stride(-1) == 1 and not any(s % per for s in t.stride()[:-1])


def mla_q4_append(c_new: torch.Tensor, r_new: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, rot: torch.Tensor,
                  start: int | torch.Tensor = 0, counts: torch.Tensor | None = None, weight: torch.Tensor | None = None) -> None:
    """Round c_new [B, T, 512] and r_new [B, T, 64] (bf16 or fp32) into positions start .. start + T - 1 of the cache,
    in place.

    ``start``: a whole number (positions past the capacity are a ValueError), or an int32 [B] device tensor, every
    sequence its own; ``counts`` int32 [B]: only sequence b's first counts[b] tokens are written.  Positions
    that a tensor puts outside the capacity are left out.  A group's scale is the power of two that puts its
    largest magnitude at 4 to 7 times itself (above 7 the next one); codes round to nearest even.  A position whose latent holds a NaN
    or an infinity is NaN to every query that sees it.  ``weight`` fp32 [B, cap]: the attention that positions have received, zeroed where one
    is written.
    """
    starts = start if isinstance(start, torch.Tensor) else None
    key = (c_new.shape, c_new.stride(), c_new.dtype, r_new.shape, r_new.stride(), r_new.dtype, packed.shape, packed.stride(),
           packed.dtype, scales.shape, scales.stride(), scales.dtype, rot.shape, rot.stride(), rot.dtype, _layout(starts), _layout(counts), _layout(weight))
    B, n, cap, c_ok, r_ok, cdt, rdt, pp, sp, rp, w_pitch = _plans.get(key) or _keep_plan(
        key, _append_plan(c_new, r_new, packed, scales, rot, starts, counts, weight))
    start0 = 0 if starts is not None else int(start)
    if starts is None and not 0 <= start0 <= start0 + n <= cap:
        raise ValueError(f"{n} tokens at position {start0} do not fit a capacity of {cap}")
    T.require_device(c_new, r_new, packed, scales, rot, starts, counts, weight)
    if T.tracked(c_new, r_new, rot, weight):
        raise ValueError("mla_q4_append carries no gradient, nor into the buffers it writes: call it under no_grad or on detached tensors")
    if B == 0 or n == 0 or cap == 0:
        return
    if not c_ok or c_new.data_ptr() % 16:
        c_new = T.contiguous_aligned(c_new)
    if not r_ok:
        r_new = r_new.contiguous()
    cs, rs = c_new.stride(), r_new.stride()
    with T.current(packed.device):
        _lib.call("k3_mla_q4_append", c_new.data_ptr(), cs[0], cs[1], cdt, r_new.data_ptr(), rs[0], rs[1], rdt, packed.data_ptr(),
                  *pp, scales.data_ptr(), *sp, rot.data_ptr(), *rp, 0 if starts is None else starts.data_ptr(), start0,
                  0 if counts is None else counts.data_ptr(), T.ptr(weight), w_pitch, B, n, cap, LATENT, ROPE, T.stream(packed))


def _append_plan(c_new, r_new, packed, scales, rot, starts, counts, weight) -> tuple:
    B, cap = _buffers(packed, scales, rot)
    if c_new.dim() != 3 or r_new.dim() != 3 or c_new.shape[2] != LATENT or r_new.shape[2] != ROPE or \
            c_new.shape[:2] != r_new.shape[:2] or c_new.shape[0] != B:
        raise ValueError(f"c_new [B, T, {LATENT}] and r_new [B, T, {ROPE}] with B = {B} expected; got {tuple(c_new.shape)}, "
                         f"{tuple(r_new.shape)}")
    cdt, rdt = T.dtype_code(c_new.dtype), T.dtype_code(r_new.dtype)
    for t, name in ((packed, "packed"), (scales, "scales"), (rot, "rot")):
        _apart(t, name)
    _per_sequence(starts, B, "start")
    _per_sequence(counts, B, "counts")
    return (B, c_new.shape[1], cap, _rows_ok(c_new, 16 // c_new.element_size()), r_new.stride(2) == 1, cdt, rdt, _pitches(packed),
            _pitches(scales), _pitches(rot), _weight_pitch(weight, B, cap))


def mla_q4_attention(q_nope: torch.Tensor, q_rot: torch.Tensor, wk: torch.Tensor, wv: torch.Tensor, packed: torch.Tensor,
                     scales: torch.Tensor, rot: torch.Tensor, scale: float, lengths: torch.Tensor | int | None = None,
                     counts: torch.Tensor | None = None, weight: torch.Tensor | None = None,
                     gate: torch.Tensor | None = None, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Absorbed latent attention of T queries of each of B sequences over the 4-bit cache -> [B, T, H, v] in out_dtype.

    q_nope [B, T, H, nope], q_rot [B, T, H, 64] (bf16 or fp32); wk [H, nope, 512], wv [H, v, 512] bf16; packed, scales,
    rot [B, cap, .].  Causal: the queries are each sequence's last T positions, query t sees positions 0 ..
    length - T + t.  ``lengths``: the sequences' lengths, a whole number for all or an int32 [B] device tensor (default: the
    capacity); ``counts`` int32 [B]: sequence b has only counts[b] queries, the first ones of its T.  A query that
    sees nothing gives zeros, whatever its gate.  A batch of more than 65,536 rows (sequences x heads) goes out in parts.

    The cache's rows are read as they lie: ``packed`` and ``rot`` 16-byte aligned with pitches of whole 16 bytes, ``scales`` 4.

    ``weight`` fp32 [B, cap], changed in place: every position's attention weight, summed over the queries and heads, is
    added to it.  ``gate`` [B, T, H * v] fp32: the output times sigmoid(gate).
    """
    length = lengths if not isinstance(lengths, torch.Tensor) else None
    if length is not None:
        lengths = None
    key = (q_nope.shape, q_nope.stride(), q_nope.dtype, q_rot.shape, q_rot.stride(), q_rot.dtype, wk.shape, wk.dtype, wv.shape, wv.dtype,
           packed.shape, packed.stride(), packed.dtype, scales.shape, scales.stride(), scales.dtype, rot.shape, rot.stride(), rot.dtype,
           _layout(lengths), _layout(counts), _layout(weight), None if gate is None else gate.shape, out_dtype)
    (B, Tq, H, V, nope, cap, qdt, code, out_code, n_ok, r_ok, pp, sp, rp, w_pitch, sizes) = _plans.get(key) or _keep_plan(
        key, _attention_plan(q_nope, q_rot, wk, wv, packed, scales, rot, lengths, counts, weight, gate, out_dtype))
    most = cap if length is None else int(length)
    if not 0 <= most <= cap:
        raise ValueError(f"length {most} outside the capacity {cap}")
    T.require_device(q_nope, q_rot, wk, wv, packed, scales, rot, weight, gate, lengths, counts)
    if T.tracked(q_nope, q_rot, wk, wv, rot, gate, weight):
        raise ValueError("mla_q4_attention carries no gradient: call it under no_grad or on detached tensors")
    device = packed.device
    out = torch.empty((B, Tq, H, V), dtype=out_dtype, device=device)
    if B == 0 or Tq == 0:
        return out
    if B > MAX_SEQUENCES or (B * H > MAX_ROWS and B > 1):
        most_at_once = max(1, min(MAX_SEQUENCES, MAX_ROWS // max(1, H)))
        for b in range(0, B, most_at_once):
            part = slice(b, min(B, b + most_at_once))
            cut = [None if t is None else t[part] for t in (lengths, counts, weight, gate)]
            out[part] = mla_q4_attention(q_nope[part], q_rot[part], wk, wv, packed[part], scales[part], rot[part], scale,
                                         most if lengths is None else cut[0], *cut[1:], out_dtype)
        return out
    if gate is not None:
        gate = T.contiguous_aligned(gate.to(torch.float32))
    if not n_ok or q_nope.data_ptr() % 16:
        q_nope = T.contiguous_aligned(q_nope.to(qdt))
    if not r_ok or q_rot.data_ptr() % 16:
        q_rot = T.contiguous_aligned(q_rot.to(qdt))
    wk, wv = T.contiguous_aligned(wk), T.contiguous_aligned(wv)
    ns, rs = q_nope.stride(), q_rot.stride()
    nbytes = _lib.size("k3_mla_q4_workspace_size", *sizes[:4], most, *sizes[4:])
    with T.current(device):
        ws = scratch(device, nbytes, "mla_q4")
        _lib.call("k3_mla_q4_attention", q_nope.data_ptr(), ns[0], ns[1], ns[2], q_rot.data_ptr(), rs[0], rs[1], rs[2], code,
                  wk.data_ptr(), wv.data_ptr(), packed.data_ptr(), *pp, scales.data_ptr(), *sp, rot.data_ptr(), *rp, T.ptr(lengths),
                  T.ptr(counts), most, B, Tq, H, LATENT, ROPE, nope, V, scale, T.ptr(gate), out.data_ptr(), out_code, T.ptr(weight),
                  w_pitch, ws.data_ptr(), ws.numel(), T.stream(packed))
    return out


def _attention_plan(q_nope, q_rot, wk, wv, packed, scales, rot, lengths, counts, weight, gate, out_dtype) -> tuple:
    B, cap = _buffers(packed, scales, rot)
    if q_nope.dim() != 4 or q_rot.dim() != 4 or q_nope.shape[:3] != q_rot.shape[:3] or q_nope.shape[0] != B or q_rot.shape[3] != ROPE:
        raise ValueError(f"q_nope [B, T, H, nope] and q_rot [B, T, H, {ROPE}] with B = {B} expected; got {tuple(q_nope.shape)}, "
                         f"{tuple(q_rot.shape)}")
    Tq, H, nope = q_nope.shape[1:]
    if wk.dim() != 3 or wv.dim() != 3 or tuple(wk.shape) != (H, nope, LATENT) or wv.shape[0] != H or wv.shape[2] != LATENT:
        raise ValueError(f"wk [{H}, {nope}, {LATENT}] and wv [{H}, v, {LATENT}] expected; got {tuple(wk.shape)}, {tuple(wv.shape)}")
    if wk.dtype != torch.bfloat16 or wv.dtype != torch.bfloat16:
        raise TypeError("wk and wv must be bfloat16 (the checkpoint dtype)")
    V = wv.shape[1]
    _per_sequence(lengths, B, "lengths")
    _per_sequence(counts, B, "counts")
    w_pitch = _weight_pitch(weight, B, cap)
    if gate is not None and (gate.numel() != B * Tq * H * V or gate.shape[:2] != (B, Tq)):
        raise ValueError(f"gate must be [{B}, {Tq}, {H * V}]; got {tuple(gate.shape)}")
    out_code = T.dtype_code(out_dtype)
    qdt = torch.bfloat16 if q_nope.dtype == torch.bfloat16 and q_rot.dtype == torch.bfloat16 else torch.float32
    sizes = (B, Tq, H, V, T.dtype_code(qdt), out_code, 0 if weight is None else 1, 0 if lengths is None else 1)
    return (B, Tq, H, V, nope, cap, qdt, T.dtype_code(qdt), out_code, q_nope.dtype == qdt and _rows_ok(q_nope, 4),
            q_rot.dtype == qdt and _rows_ok(q_rot, 4), _pitches(packed), _pitches(scales), _pitches(rot),
            w_pitch, sizes)


@dataclass
class MLACacheQ4:
    """``k3hip.mla.MLACache`` with the latents in 4 bits: packed [B, cap, 256], scales [B, cap, 16], rot [B, cap, 64], the first
    ``length`` positions valid; ``weight`` [B, cap] fp32, the attention every position has received so far, if it
    is kept (``new_cache_q4(.., weights=True)``)."""
    packed: torch.Tensor
    scales: torch.Tensor
    rot: torch.Tensor
    length: int = 0
    weight: torch.Tensor | None = None

    @property
    def capacity(self) -> int:
        return self.packed.shape[1]

    def buffers(self) -> list[torch.Tensor]:
        return [self.packed, self.scales, self.rot] + ([] if self.weight is None else [self.weight])

    def _take(self, buffers: list[torch.Tensor], length: int) -> "MLACacheQ4":
        self.packed, self.scales, self.rot = buffers[:3]
        self.weight = buffers[3] if self.weight is not None else None
        self.length = length
        return self

    def row_pitches(self) -> tuple[int, int, int]:
        """The rows' pitches of a single sequence's buffers, in elements; refuses buffers of another form."""
        B, cap = _buffers(self.packed, self.scales, self.rot)
        if B != 1:
            raise ValueError(f"a cache of {B} sequences for one sequence's token")
        _weight_pitch(self.weight, B, cap)
        if T.tracked(self.rot, self.weight):
            raise ValueError("the cache is written in place and carries no gradient: its buffers must be detached")
        return _pitches(self.packed)[1], _pitches(self.scales)[1], _pitches(self.rot)[1]

    def view(self) -> tuple[torch.Tensor, torch.Tensor]:
        """The valid prefix: latents decoded to fp32, rotary rows as they are (the kernels read the codes directly)."""
        from . import mxfp4
        B, n = self.packed.shape[0], self.length
        if B == 0 or n == 0:
            return self.packed.new_empty((B, n, LATENT), dtype=torch.float32), self.rot[:, :n]
        lat = mxfp4.decode_mxfp4(self.packed[:, :n].reshape(B * n, LATENT // 2), self.scales[:, :n].reshape(B * n, LATENT // GROUP))
        return lat.reshape(B, n, LATENT), self.rot[:, :n]

    def reserve(self, n: int) -> "MLACacheQ4":
        """Capacity for n more positions, growing as ``MLACache`` does."""
        need = self.length + n
        if need > self.capacity:
            from .mla import grown_capacity
            cap = grown_capacity(need, self.capacity)
            new = [x.new_zeros((x.shape[0], cap, *x.shape[2:])) for x in self.buffers()]
            for x, y in zip(self.buffers(), new):
                y[:, :self.length] = x[:, :self.length]
            self._take(new, self.length)
        return self

    def append(self, c_new: torch.Tensor, r_new: torch.Tensor) -> "MLACacheQ4":
        """Round T new positions into the cache, growing where it is full."""
        n = c_new.shape[1]
        self.reserve(n)
        mla_q4_append(c_new, r_new, self.packed, self.scales, self.rot, self.length, weight=self.weight)
        self.length += n
        return self

    def attend(self, q_nope: torch.Tensor, q_rot: torch.Tensor, wk: torch.Tensor, wv: torch.Tensor, scale: float,
               gate: torch.Tensor | None = None, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """``mla_q4_attention`` of the last T positions' queries over the valid prefix, its weights added to ``weight``."""
        return mla_q4_attention(q_nope, q_rot, wk, wv, self.packed, self.scales, self.rot, scale, lengths=self.length, weight=self.weight,
                                gate=gate, out_dtype=out_dtype)

    def evict(self, keep: int, sink: int = 0, recent: int = 0) -> torch.Tensor:
        """Leave min(length, keep) positions of every sequence (``k3hip.evict.cache_evict``); the capacity stays.  -> their old
        numbers [B, keep], ascending, then -1."""
        if self.weight is None:
            raise ValueError("the cache keeps no attention weights (new_cache_q4(.., weights=True))")
        from .evict import cache_evict
        new, index, _ = cache_evict(self.weight, self.buffers(), keep, lengths=self.length, sink=sink, recent=recent,
                                    capacity=max(self.capacity, keep))
        self._take(new, min(self.length, keep))
        return index

    def bytes_per_token(self) -> float:
        return sum(x.shape[2] * x.element_size() for x in (self.packed, self.scales, self.rot))

    def nbytes_used(self) -> int:
        """Bytes of the valid prefix, without the attention weights."""
        return int(self.rot.shape[0] * self.length * self.bytes_per_token())


def new_cache_q4(B: int, T: int, weights: bool = False, device="cuda") -> MLACacheQ4:
    """An empty cache for B sequences with room for T positions, rounded up as ``k3hip.mla.new_cache`` does."""
    from .mla import CACHE_STEP, _round_up
    cap = _round_up(max(T, CACHE_STEP), CACHE_STEP)
    zeros = lambda *s, dtype: torch.zeros(s, dtype=dtype, device=device)  # noqa: E731
    return MLACacheQ4(zeros(B, cap, LATENT // 2, dtype=torch.uint8), zeros(B, cap, LATENT // GROUP, dtype=torch.uint8),
                      zeros(B, cap, ROPE, dtype=torch.bfloat16), 0, zeros(B, cap, dtype=torch.float32) if weights else None)
