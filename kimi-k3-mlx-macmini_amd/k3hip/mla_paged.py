"""The paged latent cache of a batch of requests: writing it and attending over it.

The cache is a pool of pages, ``lat`` [pages, page_size, 512] and ``rot`` [pages, page_size, 64], fp16 or bf16; block tables
(``k3hip.pages``) say which pages are whose.  fp16 holds RMS-normed latents eight times finer than bf16 in the same room, and the attention
over it is faster (one term of a query or probability on the matrix cores instead of two).

``mla_paged_append`` writes new latents to their slots, RMS-normed on the way if asked for; ``mla_paged_attention`` is the absorbed latent
attention (``air_llm/models/kimi_k3/attention_mla.py:193-212``) of one token or several of every request, which reads and multiplies the pages
of a common prefix once for the whole batch.  ``MLACachePaged`` is a layer's pool beside the batch's ``PageTable``;
``k3hip.mla.MLAAttention`` runs on it.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib
from . import _torch as T
from .mla_q4 import _apart, _keep_plan, _layout, _per_sequence, _plans, scratch
from .pages import PageTable, page_shift

LATENT, ROPE, ROUND = 512, 64, 32
MAX_ROWS, MAX_SEQUENCES, MAX_LENGTH = 1 << 16, (1 << 16) - 1, 1 << 24       # heads x sequences, sequences, positions of one k3_mla_paged_attention
_CODES = {torch.float16: _lib.K3_F16, torch.bfloat16: _lib.K3_BF16}


def _steps(t: torch.Tensor) -> list[int]:
    """The strides of all dimensions but the last; of one that has a single entry: 0."""
    return [s if n > 1 else 0 for s, n in zip(t.stride()[:-1], t.shape)]


def _rows_ok(t: torch.Tensor, per: int) -> bool:
    """Contiguous rows, pitches of whole 16 bytes (``per`` elements): read as they are where the base is aligned too."""
    return t.stride(-1) == 1 and not any(s % per for s in _steps(t))


def _pool(lat, rot, least: int):
    """The pool's buffers: dtypes, shapes, row layout -> (pages, page size, dtype code, page and row pitches of both)."""
    for t, name, width in ((lat, "lat", LATENT), (rot, "rot", ROPE)):
        if t.dtype not in _CODES:
            raise TypeError(f"{name} must be float16 or bfloat16; got {t.dtype}")
        if t.dim() != 3 or t.shape[2] != width:
            raise ValueError(f"{name} must be [pages, page_size, {width}]; got {tuple(t.shape)}")
        if t.shape[0] and (t.stride(2) != 1 or (t.shape[1] > 1 and t.stride(1) < width)):
            raise ValueError(f"{name}: the values of a position must be contiguous, its rows apart (strides {t.stride()})")
    if lat.dtype != rot.dtype:
        raise TypeError(f"lat and rot must share one dtype; got {lat.dtype}, {rot.dtype}")
    if lat.shape[:2] != rot.shape[:2]:
        raise ValueError(f"lat {tuple(lat.shape)} and rot {tuple(rot.shape)} differ in pages or page size")
    pages, size = lat.shape[:2]
    page_shift(size, least)
    pitches = [(t.stride(0) if pages > 1 else 0, t.stride(1) if size > 1 and pages else t.shape[2]) for t in (lat, rot)]
    return pages, size, _CODES[lat.dtype], pitches[0], pitches[1]


def mla_paged_append(c_new: torch.Tensor, r_new: torch.Tensor, slots: torch.Tensor, lat: torch.Tensor, rot: torch.Tensor,
                     norm: torch.Tensor | None = None, eps: float = 1e-5) -> None:
    """Round c_new [B, T, 512] and r_new [B, T, 64] (bf16 or fp32) into rows ``slots`` [B, T] (int32, as ``page_tables`` gives them) of the
    pool, in place; slots outside the pool (-1) are left out, the others must differ.  ``norm`` [512]: the latents are RMS-normed first,
    norm * c / sqrt(mean(c^2) + eps).  One rounding to nearest from fp32; what exceeds fp16's largest (65,504) becomes an infinity."""
    key = (_layout(c_new), _layout(r_new), _layout(slots), _layout(lat), _layout(rot), _layout(norm), "append")
    B, n, pages, size, code, lp, rp, c_ok, r_ok, cdt, rdt = _plans.get(key) or _keep_plan(key, _append_plan(c_new, r_new, slots, lat, rot, norm))
    T.require_device(c_new, r_new, slots, lat, rot, norm)
    if T.tracked(c_new, r_new, norm, lat, rot):
        raise ValueError("mla_paged_append carries no gradient, nor into the pool it writes: call it under no_grad or on detached tensors")
    if B == 0 or n == 0 or pages == 0:
        return
    if not c_ok or c_new.data_ptr() % 16:
        c_new = T.contiguous_aligned(c_new)
    if not r_ok:
        r_new = r_new.contiguous()
    if norm is not None and (norm.dtype != torch.float32 or not norm.is_contiguous()):
        norm = norm.to(torch.float32).contiguous()
    cs, rs = _steps(c_new), _steps(r_new)
    with T.current(lat.device):
        _lib.call("k3_mla_paged_append", c_new.data_ptr(), cs[0], cs[1], cdt, r_new.data_ptr(), rs[0], rs[1], rdt, T.ptr(norm), eps,
                  slots.data_ptr(), lat.data_ptr(), *lp, rot.data_ptr(), *rp, code, pages, size, B, n, LATENT, ROPE, T.stream(lat))


def _append_plan(c_new, r_new, slots, lat, rot, norm) -> tuple:
    pages, size, code, lp, rp = _pool(lat, rot, 1)
    for t, name in ((lat, "lat"), (rot, "rot")):
        _apart(t, name)
    if c_new.dim() != 3 or r_new.dim() != 3 or c_new.shape[2] != LATENT or r_new.shape[2] != ROPE or c_new.shape[:2] != r_new.shape[:2]:
        raise ValueError(f"c_new [B, T, {LATENT}] and r_new [B, T, {ROPE}] expected; got {tuple(c_new.shape)}, {tuple(r_new.shape)}")
    if slots.dtype != torch.int32:
        raise TypeError(f"slots must be an int32 tensor; got {slots.dtype}")
    B, n = c_new.shape[:2]
    if tuple(slots.shape) != (B, n) or not slots.is_contiguous():
        raise ValueError(f"slots must be a contiguous [{B}, {n}]; got {tuple(slots.shape)}")
    if norm is not None and tuple(norm.shape) != (LATENT,):
        raise ValueError(f"norm must be [{LATENT}]; got {tuple(norm.shape)}")
    cdt, rdt = T.dtype_code(c_new.dtype), T.dtype_code(r_new.dtype)
    return (B, n, pages, size, code, lp, rp, _rows_ok(c_new, 16 // c_new.element_size()), r_new.stride(2) == 1, cdt, rdt)


def mla_paged_attention(q_nope: torch.Tensor, q_rot: torch.Tensor, wk: torch.Tensor, wv: torch.Tensor, lat: torch.Tensor, rot: torch.Tensor,
                        table: torch.Tensor, lengths: torch.Tensor, scale: float, counts: torch.Tensor | None = None,
                        prefix: torch.Tensor | None = None, gate: torch.Tensor | None = None, out_dtype: torch.dtype = torch.float32,
                        max_length: int | None = None) -> torch.Tensor:
    """Absorbed latent attention of T queries of each of B sequences over the pool's pages -> [B, T, H, v] in out_dtype.

    q_nope [B, T, H, nope], q_rot [B, T, H, 64] (bf16 or fp32); wk [H, nope, 512], wv [H, v, 512] bf16; lat, rot [pages, page_size, .], a page
    size from 32 on; table int32 [B, blocks]: position j of sequence b lies in page table[b, j // page_size].  Causal: the queries are each
    sequence's last positions; with n = counts[b] (int32 [B], default T) query t < n sees positions 0 .. lengths[b] - n + t, and
    later ones see nothing.  ``lengths`` int32 [B] on the device; ``max_length``: none is longer (default: what the table holds; longer ones
    are cut).  A query that sees nothing gives zeros, whatever its gate; a position on a page outside the pool counts as not there.

    ``prefix`` int32 [n]: the pages of the first n * page_size positions of every sequence, read and multiplied once for the whole batch;
    ``table`` counts from position 0 all the same, its first n columns are not read.

    ``gate`` [B, T, H * v] fp32: the output times sigmoid(gate).  A batch of more than 65,536 rows (sequences x heads) goes out in parts.
    """
    key = (q_nope.shape, q_nope.stride(), q_nope.dtype, q_rot.shape, q_rot.stride(), q_rot.dtype, wk.shape, wk.dtype, wv.shape, wv.dtype,
           lat.shape, lat.stride(), lat.dtype, rot.shape, rot.stride(), rot.dtype, _layout(table), _layout(lengths), _layout(counts), _layout(prefix),
           None if gate is None else gate.shape, out_dtype, max_length)
    (B, Tq, H, V, nope, pages, size, code, lp, rp, blocks, pitch, n_prefix, most, qdt, q_code, out_code, n_ok, r_ok, sizes) = _plans.get(
        key) or _keep_plan(key, _attention_plan(q_nope, q_rot, wk, wv, lat, rot, table, lengths, counts, prefix, gate, out_dtype, max_length))
    T.require_device(q_nope, q_rot, wk, wv, lat, rot, table, lengths, counts, prefix, gate)
    if T.tracked(q_nope, q_rot, wk, wv, lat, rot, gate):
        raise ValueError("mla_paged_attention carries no gradient: call it under no_grad or on detached tensors")
    device = lat.device
    out = torch.empty((B, Tq, H, V), dtype=out_dtype, device=device)
    if B == 0 or Tq == 0:
        return out
    if B > MAX_SEQUENCES or (B * H > MAX_ROWS and B > 1):
        most_at_once = max(1, min(MAX_SEQUENCES, MAX_ROWS // max(1, H)))
        for b in range(0, B, most_at_once):
            part = slice(b, min(B, b + most_at_once))
            out[part] = mla_paged_attention(q_nope[part], q_rot[part], wk, wv, lat, rot, table[part], lengths[part], scale,
                                            None if counts is None else counts[part], prefix, None if gate is None else gate[part], out_dtype,
                                            max_length)
        return out
    if gate is not None:
        gate = T.contiguous_aligned(gate.to(torch.float32))
    if not n_ok or q_nope.data_ptr() % 16:
        q_nope = T.contiguous_aligned(q_nope.to(qdt))
    if not r_ok or q_rot.data_ptr() % 16:
        q_rot = T.contiguous_aligned(q_rot.to(qdt))
    wk, wv = T.contiguous_aligned(wk), T.contiguous_aligned(wv)
    ns, rs = _steps(q_nope), _steps(q_rot)
    nbytes = _lib.size("k3_mla_paged_workspace_size", *sizes)
    with T.current(device):
        ws = scratch(device, nbytes, "mla_paged")
        _lib.call("k3_mla_paged_attention", q_nope.data_ptr(), ns[0], ns[1], ns[2], q_rot.data_ptr(), rs[0], rs[1], rs[2], q_code, wk.data_ptr(),
                  wv.data_ptr(), lat.data_ptr(), *lp, rot.data_ptr(), *rp, code, pages, size, table.data_ptr(), pitch, blocks, T.ptr(prefix),
                  n_prefix, lengths.data_ptr(), T.ptr(counts), most, B, Tq, H, LATENT, ROPE, nope, V, scale, T.ptr(gate), out.data_ptr(), out_code,
                  ws.data_ptr(), ws.numel(), T.stream(lat))
    return out


def _attention_plan(q_nope, q_rot, wk, wv, lat, rot, table, lengths, counts, prefix, gate, out_dtype, max_length) -> tuple:
    pages, size, code, lp, rp = _pool(lat, rot, ROUND)
    for t, name, pitches in ((lat, "lat", lp), (rot, "rot", rp)):
        if pages and (pitches[0] % 8 or pitches[1] % 8):
            raise ValueError(f"{name}: rows are read as they lie, with pitches of whole 16 bytes; got strides {t.stride()}")
    if q_nope.dim() != 4 or q_rot.dim() != 4 or q_nope.shape[:3] != q_rot.shape[:3] or q_rot.shape[3] != ROPE:
        raise ValueError(f"q_nope [B, T, H, nope] and q_rot [B, T, H, {ROPE}] expected; got {tuple(q_nope.shape)}, {tuple(q_rot.shape)}")
    B, Tq, H, nope = q_nope.shape
    if wk.dim() != 3 or wv.dim() != 3 or tuple(wk.shape) != (H, nope, LATENT) or wv.shape[0] != H or wv.shape[2] != LATENT:
        raise ValueError(f"wk [{H}, {nope}, {LATENT}] and wv [{H}, v, {LATENT}] expected; got {tuple(wk.shape)}, {tuple(wv.shape)}")
    if wk.dtype != torch.bfloat16 or wv.dtype != torch.bfloat16:
        raise TypeError("wk and wv must be bfloat16 (the checkpoint dtype)")
    V = wv.shape[1]
    if table.dtype != torch.int32:
        raise TypeError(f"table must be an int32 tensor; got {table.dtype}")
    if table.dim() != 2 or table.shape[0] != B or (table.shape[1] > 1 and table.stride(1) != 1) or (B > 1 and table.stride(0) < table.shape[1]):
        raise ValueError(f"table must be [{B}, blocks] with contiguous rows; got {tuple(table.shape)}, strides {table.stride()}")
    if lengths is None:
        raise ValueError("lengths must be an int32 tensor")
    _per_sequence(lengths, B, "lengths")
    _per_sequence(counts, B, "counts")
    n_prefix = 0
    if prefix is not None:
        if prefix.dtype != torch.int32:
            raise TypeError(f"prefix must be an int32 tensor; got {prefix.dtype}")
        if prefix.dim() != 1 or not prefix.is_contiguous():
            raise ValueError(f"prefix must be a contiguous [pages]; got {tuple(prefix.shape)}")
        n_prefix = prefix.shape[0]
    blocks = table.shape[1]
    most = min(blocks * size, MAX_LENGTH)
    if max_length is not None:
        if not 0 <= int(max_length) <= blocks * size:
            raise ValueError(f"max_length {max_length} outside the table's {blocks} x {size} positions")
        most = int(max_length)
    if gate is not None and (gate.numel() != B * Tq * H * V or gate.shape[:2] != (B, Tq)):
        raise ValueError(f"gate must be [{B}, {Tq}, {H * V}]; got {tuple(gate.shape)}")
    out_code = T.dtype_code(out_dtype)
    qdt = torch.bfloat16 if q_nope.dtype == torch.bfloat16 and q_rot.dtype == torch.bfloat16 else torch.float32
    n_ok, r_ok = q_nope.dtype == qdt and _rows_ok(q_nope, 4), q_rot.dtype == qdt and _rows_ok(q_rot, 4)
    return (B, Tq, H, V, nope, pages, size, code, lp, rp, blocks, table.stride(0) if B > 1 else blocks, n_prefix, most, qdt, T.dtype_code(qdt),
            out_code, n_ok, r_ok, (B, Tq, H, most, n_prefix * size, code, out_code))


@dataclass
class MLACachePaged:
    """One layer's pool of pages, ``latent`` [pages, page_size, 512] and ``rot`` [pages, page_size, 64], beside the batch's tables, which all
    layers share: ``pages.extend(..)`` once a step, then every layer."""
    pages: PageTable
    latent: torch.Tensor
    rot: torch.Tensor

    def append(self, c_new: torch.Tensor, r_new: torch.Tensor, norm: torch.Tensor | None = None, eps: float = 1e-5) -> "MLACachePaged":
        """Write the tokens of the step, [batch, T, .], to their slots."""
        if c_new.shape[:2] != self.pages.slots.shape:
            raise ValueError(f"{tuple(c_new.shape[:2])} new tokens for slots of {tuple(self.pages.slots.shape)}: call pages.extend for the step first")
        mla_paged_append(c_new, r_new, self.pages.slots, self.latent, self.rot, norm, eps)
        return self

    def attend(self, q_nope: torch.Tensor, q_rot: torch.Tensor, wk: torch.Tensor, wv: torch.Tensor, scale: float,
               gate: torch.Tensor | None = None, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """``mla_paged_attention`` of the step's tokens over all that their requests hold."""
        p = self.pages
        return mla_paged_attention(q_nope, q_rot, wk, wv, self.latent, self.rot, p.table, p.lengths, scale, counts=p.counts, prefix=p.prefix,
                                   gate=gate, out_dtype=out_dtype)

    def bytes_per_token(self) -> float:
        return sum(x.shape[2] * x.element_size() for x in (self.latent, self.rot))


def new_cache_paged(pages: PageTable, dtype: torch.dtype = torch.float16) -> MLACachePaged:
    """A layer's empty pool for the tables' pages."""
    if dtype not in _CODES:
        raise TypeError(f"the pool must be float16 or bfloat16; got {dtype}")
    page_shift(pages.page_size, ROUND)
    zeros = lambda w: torch.zeros((pages.pages, pages.page_size, w), dtype=dtype, device=pages.table.device)  # noqa: E731
    return MLACachePaged(pages, zeros(LATENT), zeros(ROPE))
