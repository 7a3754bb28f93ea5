"""Block tables and slot maps of a serving step, built on the device from request lengths.

`PagePool` keeps a request's pages on the host and a forward copies its table over
(`PagedPackedCache`, `DeviceTable`).  Here the batch's tables, lengths and free pages live on the
device: one launch (`wtq_plan_tokens`) turns the lengths and the numbers of new tokens into each
token's sequence, position and slot, takes the pages the step needs, writes them to the table
and, for drafted trees, works out depths and ancestor masks, without the host waiting for
anything.  `DevicePages` is that state over pages a `PagePool` lends: they stay reserved there
under one owner, with its fences, until `close()`.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib
from .page_pool import PagePool, PoolExhausted, StalePage


class TokenPlan(NamedTuple):
    """What a step's kernels read.  Entries past the last token are -1 (`slot_ends` 0)."""

    seq_lens: torch.Tensor        # (B,) int32, with the new tokens
    held: torch.Tensor            # (B,) int32 pages of each sequence's row of the table
    free_count: torch.Tensor      # (1,) int32
    starts: torch.Tensor          # (B + 1,) int32 first token of each sequence
    sequence: torch.Tensor        # (T,) int32
    positions: torch.Tensor       # (T,) int32; in a tree: the length plus the depth, -1 for padding
    slot_pages: torch.Tensor      # (T, 1) int32 page of each token: the page table of a one-token sequence
    slot_ends: torch.Tensor       # (T,) int32 slot + 1: that sequence's length
    mask: torch.Tensor | None     # (B, Q, ceil(Q / 32)) int32 words, with parents


def _int32(name: str, t: torch.Tensor, *shape: int) -> torch.Tensor:
    if t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous int32 {shape}, got {t.dtype} {tuple(t.shape)}")
    return t


def plan_tokens(lengths, new_tokens, table, held, free_pages, free_count, page_size: int, tokens: int, *,
                parents=None, out: TokenPlan | None = None, ticket=None, status=None) -> TokenPlan:
    """Grant `new_tokens[b]` more tokens to every sequence, all or none.

    lengths, new_tokens, held (B,) int32; table (B, W) int32 with contiguous rows, whose first held[b]
    entries are sequence b's pages: entries behind them are written in place, and the pages come off the
    end of the first free_count[0] entries of `free_pages`, in batch order.  `tokens`: room of the
    per-token results (the sum of new_tokens, or more).  With `parents` (B, Q) int32, every sequence
    gets a tree of Q tokens, `new_tokens` is None and tokens = B * Q: the parent of each token within its
    tree, before it; -1 below the history's last token, -2 for padding.  A step that the free pages or
    the table's width do not cover takes nothing and sets `STATUS_NO_PAGES` in `status`.

    The state comes back as new tensors, or goes to those of `out`; those may be the inputs
    (lengths as seq_lens, held, free_count), with `ticket`, an int32 word that is zero, and share no memory otherwise.
    """
    tree = parents is not None
    if tree == (new_tokens is not None):
        raise ValueError("plan_tokens needs new_tokens or parents, and not both")
    if out is None or ticket is not None:
        got = _lib.host().plan(lengths, new_tokens, table, held, free_pages, free_count, int(page_size), int(tokens),
                               parents, None if out is None else tuple(out), ticket, status)
        if got is not None:
            return TokenPlan(*got)
    dev = _lib.require_cuda(lengths, table, held, free_pages, free_count, parents if tree else new_tokens)
    _lib.reachable("status", status, dev)
    _lib.reachable("ticket", ticket, dev)
    if table.dim() != 2 or table.dtype != torch.int32 or table.stride(1) != 1 or table.shape[1] < 1:
        raise ValueError("table must be int32 (B, width) with contiguous rows")
    B, W = table.shape
    if page_size < 1 or tokens < 0:
        raise ValueError("page_size must be positive and tokens not negative")
    _int32("lengths", lengths, B)
    _int32("held", held, B)
    _int32("free_pages", free_pages, free_pages.numel())
    _int32("free_count", free_count, 1)
    Q = 0
    if tree:
        if parents.dim() != 2 or parents.shape[0] != B or parents.dtype != torch.int32 or parents.shape[1] < 1 \
                or (parents.stride(1) != 1 and parents.shape[1] > 1):
            raise ValueError("parents must be int32 (B, Q) with contiguous rows")
        Q = parents.shape[1]
        if tokens != B * Q:
            raise ValueError(f"trees of {Q} tokens for {B} sequences are {B * Q} tokens, not {tokens}")
    else:
        _int32("new_tokens", new_tokens, B)
    if B > 1 and table.stride(0) < W:
        raise ValueError("table rows overlap")
    if out is None:
        empty = lambda *shape: torch.empty(shape, dtype=torch.int32, device=dev)       # noqa: E731
        out = TokenPlan(empty(B), empty(B), empty(1), empty(B + 1), empty(tokens), empty(tokens), empty(tokens, 1),
                        empty(tokens), empty(B, Q, -(-Q // 32)) if tree else None)
    else:
        for name, t, shape in (("seq_lens", out.seq_lens, (B,)), ("held", out.held, (B,)),
                               ("free_count", out.free_count, (1,)), ("starts", out.starts, (B + 1,)),
                               ("sequence", out.sequence, (tokens,)), ("positions", out.positions, (tokens,)),
                               ("slot_pages", out.slot_pages, (tokens, 1)), ("slot_ends", out.slot_ends, (tokens,)),
                               *((("mask", out.mask, (B, Q, -(-Q // 32))),) if tree else ())):
            if t is None or t.device != dev:
                raise ValueError(f"out.{name} must be on {dev}")
            _int32(f"out.{name}", t, *shape)
        if ticket is not None:
            _int32("ticket", ticket, 1)
    words = _lib.Plan(*(None if t is None else t.data_ptr() for t in out))
    ptr = lambda t: None if t is None else t.data_ptr()                                # noqa: E731
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().wtq_plan_tokens(
            lengths.data_ptr(), ptr(new_tokens), ptr(parents), parents.stride(0) if tree else 0, table.data_ptr(),
            table.stride(0), held.data_ptr(), free_pages.data_ptr(), free_count.data_ptr(), B, W, int(page_size),
            int(tokens), Q, free_pages.numel(), ctypes.byref(words), ptr(ticket), ptr(status), _lib.stream_ptr(dev)))
    return out


class DevicePages:
    """A batch's page table, lengths and free pages on the device.

    `pages` pages of `pool` are reserved under `owner` and dealt out from here; `batch` sequences of at
    most `width` pages each.  `extend` appends to sequences, `keep` shortens them after a drafted step,
    `release` ends some of them; each is launches on the current stream and waits for nothing.  `table`
    and `lengths` are what the append and attention calls read.  What a launch refuses is collected in
    `status`; `check()` synchronises and raises.
    """

    def __init__(self, pool: PagePool, owner: str, *, pages: int, batch: int, width: int):
        if pool.device.type != "cuda":
            raise _lib.BackendError("DevicePages needs a pool on a CUDA device; there is no CPU path")
        self.pool, self.owner, self.page_size = pool, owner, pool.page_size
        if pool.held(owner):
            raise ValueError(f"{owner!r} already holds pages")
        ids = [ref.page for ref in pool.ensure(owner, pages * pool.page_size)]
        self._reservation = pool.reservation(owner)
        dev = pool.device
        self.free_pages = torch.tensor(ids[::-1], dtype=torch.int32, device=dev)
        self.free_count = torch.tensor([len(ids)], dtype=torch.int32, device=dev)
        self.table = torch.full((batch, width), -1, dtype=torch.int32, device=dev)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.held = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)
        self._ticket = torch.zeros(1, dtype=torch.int32, device=dev)
        self._room: dict = {}

    def ensure_held(self) -> None:
        """Raise `StalePage` once the pages have been given back (`close`, or a release of the owner in the pool):
        they may be another request's by then."""
        if self.pool.reservation(self.owner) is not self._reservation:
            raise StalePage(f"{self.owner!r} no longer holds the pages of this batch")

    def extend(self, new_tokens=None, *, tokens: int | None = None, parents=None) -> TokenPlan:
        """Append new_tokens[b] tokens (`tokens` in all, or room for more), or a tree each.  The plan's
        per-token tensors are this object's own and written again by a later call for about as many
        tokens; its state tensors are `lengths`, `held`, `free_count`."""
        self.ensure_held()
        B = self.lengths.numel()
        if parents is not None:
            Q = int(parents.shape[1]) if parents.dim() == 2 else 0
            tokens = B * Q
        elif tokens is None:
            raise ValueError("extend needs the number of tokens: reading it off the device would wait")
        else:
            Q = 0
        # (a captured step keeps its addresses: rooms are never given up, so there is one a power of two)
        size = tokens if Q else 1 << max(tokens - 1, 0).bit_length()
        room = self._room.get((size, Q))
        if room is None:
            e = lambda *shape: torch.empty(shape, dtype=torch.int32, device=self.pool.device)   # noqa: E731
            room = self._room[(size, Q)] = TokenPlan(
                self.lengths, self.held, self.free_count, e(B + 1), e(size), e(size), e(size, 1), e(size),
                e(B, Q, -(-Q // 32)) if Q else None)
        if size != tokens:
            room = room._replace(**{name: getattr(room, name)[:tokens]
                                    for name in ("sequence", "positions", "slot_pages", "slot_ends")})
        return plan_tokens(self.lengths, new_tokens, self.table, self.held, self.free_pages, self.free_count,
                           self.page_size, tokens, parents=parents, out=room, ticket=self._ticket, status=self.status)

    def keep(self, keep: torch.Tensor, counts: torch.Tensor, drafted: int, plan: TokenPlan | None = None) -> torch.Tensor:
        """Of the last `drafted` tokens of every sequence, keep token keep[b][i] as its i-th for
        i < counts[b], in every layer of the pool, and shorten `lengths` (`keep_tokens`).  With the step's
        `plan`, a step that was refused leaves everything as it is."""
        from .packed_backend import keep_tokens
        pool = self.pool
        if pool.dense:
            raise ValueError("keep serves packed pools")
        self.ensure_held()
        after = keep_tokens(pool.k_pages, pool.k_norms, pool.v_pages, pool.v_norms, self.table, self.lengths, keep,
                            counts, drafted, granted=None if plan is None else plan.starts[-1:], status=self.status)
        self.lengths.copy_(after)
        return self.lengths

    def release(self, marks: torch.Tensor) -> None:
        """End the sequences with marks[b] != 0: their pages are free for the next `extend`."""
        self.ensure_held()
        dev = _lib.require_cuda(marks, self.table)
        _int32("marks", marks, self.lengths.numel())
        with torch.cuda.device(dev):
            _lib.check(_lib.lib().wtq_release_tokens(
                marks.data_ptr(), self.table.data_ptr(), self.table.stride(0), self.lengths.data_ptr(),
                self.held.data_ptr(), self.free_pages.data_ptr(), self.free_count.data_ptr(), self.lengths.numel(),
                self.table.shape[1], self.free_pages.numel(), self.status.data_ptr(), _lib.stream_ptr(dev)))

    def check(self) -> None:
        """Raise if a launch since the last check refused something (synchronises)."""
        word = int(self.status.item())
        if not word:
            return
        self.status.zero_()
        if word & _lib.STATUS_NO_PAGES:
            raise PoolExhausted("a step needed more pages than are free, or than a row of the table has room for; "
                                "it was not granted")
        raise StalePage(f"the kernels refused part of the batch (status {word:#x}: bit {_lib.STATUS_BAD_PAGE} page id "
                        f"outside the pool, bit {_lib.STATUS_BAD_POSITION} position or path out of range, bit "
                        f"{_lib.STATUS_BAD_PARENT} parent behind its child)")

    def close(self, fence=None) -> int:
        """Give all pages back to the pool, behind a fence; calls that would use them after that raise `StalePage`."""
        if self.pool.reservation(self.owner) is not self._reservation:
            return 0                                       # (given back already; the name may be another's)
        return self.pool.release(self.owner, fence)
