"""Pages of a cache that a batch of requests shares: block tables, the list of free pages, the rows that new tokens go to.

``page_tables`` changes the lengths of all requests at once, on the device: requests that grow take pages from the list of free
ones, requests that shrink or end give theirs back, and every new token gets its row in the pool ("slot").  Nothing comes to the host, so a
step can be captured into a graph.  ``PageTable`` keeps the tables of a batch; the layers' caches (``k3hip.mla_paged.MLACachePaged``) share
one.  The reference's cache is one sequence's, contiguous (``air_llm/models/kimi_k3/attention_mla.py:62-117``).
"""
from __future__ import annotations

import torch

from . import _lib
from . import _torch as T
from .mla_q4 import _keep_plan, _layout, _per_sequence, _plans, scratch

MAX_PAGE = 1 << 16


def page_shift(page_size: int, least: int = 1) -> int:
    """log2 of a page size; refuses what is no power of two from ``least`` to 65,536."""
    page_size = int(page_size)
    if not least <= page_size <= MAX_PAGE or page_size & (page_size - 1):
        raise ValueError(f"page_size {page_size} must be a power of two, {least} to {MAX_PAGE}")
    return page_size.bit_length() - 1


def page_tables(table: torch.Tensor, lengths: torch.Tensor, target: torch.Tensor, free: torch.Tensor, used: torch.Tensor, page_size: int,
                tokens: int = 0, shared: torch.Tensor | None = None, inplace: bool = False):
    """-> (lengths [B], used [1], slots [B, tokens]), int32: what the requests hold now, how many entries of the list are taken, and the
    rows of the new tokens.

    All int32 device tensors.  ``table`` [B, blocks]: request b's pages, in order, ceil(lengths[b] / page_size) of them; changed in
    place.  ``target`` [B]: the lengths to come to (negative: 0).  ``free`` [pages]: its entries from ``used`` [1] on are the pages that nobody
    holds; changed in place, where pages are given back.  ``shared`` [B]: so many of a request's first pages are not its own and are never
    given back; changed in place: a request that has come below them and grows again takes pages of its own in their places, and its entry comes down to
    what is left of them.  ``inplace``: ``lengths`` and ``used`` are written over instead of new tensors.

    Pages given back come in front of the list's free entries, in the batch's order, and can be taken in the same call.  Pages are taken
    in the batch's order; from the first request on that there are not enough for, requests that need pages stay at their length, as does one whose
    target the table has no room for.  slots[b, i] = page * page_size + position % page_size of request b's i-th new token, -1 past its new length.
    """
    key = (_layout(table), _layout(lengths), _layout(target), _layout(free), _layout(used), _layout(shared), page_size, tokens, "tables")
    B, blocks, pages, pitch, page_size, tokens, nbytes = _plans.get(key) or _keep_plan(
        key, _tables_plan(table, lengths, target, free, used, shared, page_size, tokens))
    T.require_device(table, lengths, target, free, used, shared)
    new_lengths, new_used = (lengths, used) if inplace else (torch.empty_like(lengths), torch.empty_like(used))
    slots = lengths.new_empty((B, tokens))
    if B == 0:
        if not inplace:
            new_used.copy_(used)
        return new_lengths, new_used, slots
    with T.current(table.device):
        ws = scratch(table.device, nbytes, "page_tables")
        _lib.call("k3_page_tables", table.data_ptr(), pitch, blocks, lengths.data_ptr(), target.data_ptr(), T.ptr(shared), free.data_ptr(), pages,
                  used.data_ptr(), page_size, B, tokens, new_lengths.data_ptr(), new_used.data_ptr(), slots.data_ptr(), ws.data_ptr(), ws.numel(),
                  T.stream(table))
    return new_lengths, new_used, slots


def _tables_plan(table, lengths, target, free, used, shared, page_size, tokens) -> tuple:
    page_shift(page_size)
    tokens = int(tokens)
    if tokens < 0:
        raise ValueError(f"tokens {tokens} must not be negative")
    if table.dtype != torch.int32 or free.dtype != torch.int32:
        raise TypeError(f"table and free must be int32 tensors; got {table.dtype}, {free.dtype}")
    if table.dim() != 2 or (table.shape[1] > 1 and table.stride(1) != 1):
        raise ValueError(f"table must be [B, blocks] with contiguous rows; got {tuple(table.shape)}, strides {table.stride()}")
    B, blocks = table.shape
    if B > 1 and table.stride(0) < blocks:
        raise ValueError(f"table: the requests' rows overlap in memory (strides {table.stride()}); they are written")
    if free.dim() != 1 or not free.is_contiguous():
        raise ValueError(f"free must be a contiguous [pages]; got {tuple(free.shape)}")
    for t, name in ((lengths, "lengths"), (target, "target"), (shared, "shared")):
        _per_sequence(t, B, name)
    _per_sequence(used, 1, "used")
    return (B, blocks, free.shape[0], table.stride(0) if B > 1 else blocks, int(page_size), tokens, _lib.size("k3_page_tables_workspace_size", B))


class PageTable:
    """The block tables of ``batch`` requests of up to ``capacity`` positions over ``pages`` pages.

    ``extend`` takes what the next tokens need and keeps, for the layers of the step, their rows (``slots`` [batch, tokens]), how many
    every request got (``counts``) and the new ``lengths``; all on the device."""

    def __init__(self, batch: int, capacity: int, pages: int, page_size: int = 64, device="cuda"):
        page_shift(page_size)
        whole = lambda *s: torch.zeros(s, dtype=torch.int32, device=device)  # noqa: E731
        self.page_size, self.pages = int(page_size), int(pages)
        self.table = whole(batch, -(-int(capacity) // self.page_size)) - 1
        self.lengths, self.counts, self.used = whole(batch), whole(batch), whole(1)
        self.shared = None                      # [batch]: pages of the common prefix that a request's row begins with
        self.free = torch.arange(self.pages, dtype=torch.int32, device=device)
        self.prefix = None                      # the common prefix's pages
        self.slots = whole(batch, 0)

    @property
    def batch(self) -> int:
        return self.table.shape[0]

    @property
    def capacity(self) -> int:
        return self.table.shape[1] * self.page_size

    def resize(self, target: torch.Tensor, tokens: int = 0) -> torch.Tensor:
        """All requests to ``target`` [batch] int32 positions -> slots of up to ``tokens`` new tokens each (``page_tables``).  None goes below
        a common prefix.  One that grows by more than ``tokens`` has slots of the first ones only: the rest, on the pages of its row, is
        the caller's to write before anything attends (``extend`` gives none more than it has slots)."""
        _per_sequence(target, self.batch, "target")
        if self.prefix is not None:
            target = target.clamp(min=len(self.prefix) * self.page_size)
        before = self.lengths.clone()
        _, _, self.slots = page_tables(self.table, self.lengths, target, self.free, self.used, self.page_size, tokens, self.shared, inplace=True)
        self.counts = (self.lengths - before).clamp_(min=0)
        return self.slots

    def extend(self, counts: int | torch.Tensor, tokens: int | None = None) -> torch.Tensor:
        """Room for ``counts`` more tokens of every request (a number, or int32 [batch], 0 for a request that rests, below 0 for one that gives
        so many back) -> slots [batch, tokens] (``tokens``: the most that a request gets; needed for a tensor, whose larger entries are cut to
        it).  A request for which there is no page left gets none: its ``counts`` entry is 0, its slots are -1."""
        if isinstance(counts, torch.Tensor):
            _per_sequence(counts, self.batch, "counts")
            if tokens is None:
                raise ValueError("tokens: the most new tokens of a request, where counts is a tensor")
            tokens = int(tokens)
            counts = counts.clamp(max=tokens)
        else:
            tokens = max(int(counts), 0) if tokens is None else int(tokens)
            if counts > tokens:
                raise ValueError(f"{counts} new tokens of every request for {tokens} slots of each")
        if tokens >= (1 << 31) - self.capacity:         # (lengths are int32)
            raise ValueError(f"{tokens} new tokens of a request and the {self.capacity} it may hold do not fit 32 bits")
        return self.resize(self.lengths + counts, tokens)

    def truncate(self, lengths: torch.Tensor) -> None:
        """No request longer than ``lengths`` [batch] int32; pages behind that are given back.  A common prefix stays."""
        _per_sequence(lengths, self.batch, "lengths")
        self.resize(torch.minimum(self.lengths, lengths))

    def release(self, ended: torch.Tensor) -> None:
        """The requests where ``ended`` [batch] bool is true give back all pages of their own: they hold nothing, or the common prefix."""
        if tuple(ended.shape) != (self.batch,) or ended.dtype != torch.bool:
            raise ValueError(f"ended must be a bool [{self.batch}]; got {ended.dtype} {tuple(ended.shape)}")
        self.truncate(torch.where(ended, torch.zeros_like(self.lengths), self.lengths))

    def share(self, length: int, source: int = 0) -> None:
        """Make the first ``length`` positions of request ``source``, whole pages, the common prefix of the batch: all others, which must
        hold nothing yet, and whatever takes their places later, begin with them.  The pages stay taken.
        Reads the lengths on the host.  A graph that was captured before does not know of the prefix: capture its steps anew."""
        n, left = divmod(int(length), self.page_size)
        if left or not 0 < n <= self.table.shape[1]:
            raise ValueError(f"a prefix of {length} positions is not 1 to {self.table.shape[1]} whole pages of {self.page_size}")
        if self.prefix is not None:
            raise ValueError("the batch has a common prefix already")
        if not 0 <= source < self.batch:
            raise ValueError(f"source {source} outside the batch of {self.batch}")
        held = self.lengths.tolist()
        if held[source] < length:
            raise ValueError(f"request {source} holds {held[source]} positions, the prefix {length}")
        if any(h for b, h in enumerate(held) if b != source):
            raise ValueError("the other requests must hold nothing when a prefix is shared")
        self.prefix = self.table[source, :n].clone()
        self.table[:, :n] = self.prefix
        self.lengths.clamp_(min=int(length))
        self.shared = torch.full_like(self.lengths, n)
