"""Copies of cache pages, in the tensors of all layers at once.

A request that is forked shares its whole pages with its children and copies the page that it has begun; a cache that is made
compact moves whole pages.  A move (source, target, n) makes slots 0 .. n - 1 of page ``target`` those of page ``source``; every
other slot stays as it is.  The moves of one call happen as if at once: no page is written twice, and none that is written is
read (calls that ask for it are refused).
"""
from __future__ import annotations

from typing import Sequence, Union

import torch

from . import ops
from .build import load_entry_points
from .ops import KernelError

_MOVES_OF_A_LAUNCH = 2048
_REFUSED = {-10: "a move names a page outside the pool, or more slots than a page has",
            -11: "a page is the target of two moves, or of one and the source of another",
            -12: "no memory on the host to check the moves"}


class PageCopier:
    """Copies pages of ``tensors``, the keys and values of any number of layers: contiguous [pages, heads, page_size, dim] on one
    device, all with as many pages of as many slots; heads, dims and dtypes (of 2 or 4 bytes) may differ.  Made once with the cache;
    it keeps the tensors alive and their addresses on the device."""

    def __init__(self, tensors: Sequence[torch.Tensor]):
        self._tensors = list(tensors)
        if not self._tensors:
            raise KernelError("a page copier needs the tensors whose pages it copies")
        first = self._tensors[0]
        for t in self._tensors:
            if t.dim() != 4 or not t.is_contiguous() or 0 in t.shape:
                raise KernelError("page copies take contiguous tensors [pages, heads, page_size, dim]")
            if t.element_size() not in (2, 4):
                raise KernelError(f"dtype {t.dtype} is not supported (elements of 2 and 4 bytes are)")
            if t.shape[0] != first.shape[0] or t.shape[2] != first.shape[2] or t.device != first.device:
                raise KernelError("the tensors of a page copier have as many pages of as many slots, on one device")
        spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in self._tensors)
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise KernelError("the tensors of a page copier must not overlap")
        self.pages, self.page_size = first.shape[0], first.shape[2]
        self._page_bytes = max(t[0].numel() * t.element_size() for t in self._tensors)
        if self._page_bytes > 1 << 30:
            raise KernelError(f"pages of {self._page_bytes} bytes are refused: up to {1 << 30}")
        ops._cuda(*self._tensors)
        table = []
        for t in self._tensors:
            row = t.shape[3] * t.element_size()
            # (two 32-bit numbers in each of the last two)
            table.append([t.data_ptr(), t[0].numel() * t.element_size(), (row << 32) | row * t.shape[2], t.shape[1]])
        align = 0
        for address, _, rows, _ in table:
            align |= address | rows >> 32
        self._vector = next(v for v in (16, 4, 2) if align % v == 0)
        self._table = torch.tensor(table, dtype=torch.int64).to(first.device)
        torch.cuda.synchronize(first.device)                 # (whatever stream copies first finds the table)
        self._entry = load_entry_points("pages.cu").b200_copy_pages

    def copy(self, moves: Union[torch.Tensor, Sequence[Sequence[int]]]) -> None:
        """``moves``: (source, target, slots) each, as a sequence or an int32 tensor [n, 3] on the host, read before this returns.  The
        copies run on the current stream (a captured graph holds the moves that it was captured with)."""
        if not isinstance(moves, torch.Tensor):
            moves = torch.tensor([tuple(m) for m in moves], dtype=torch.int32).reshape(-1, 3)
        if moves.dtype != torch.int32 or moves.dim() != 2 or moves.shape[1] != 3 or moves.is_cuda or not moves.is_contiguous():
            raise KernelError("moves are int32 [n, 3] on the host: source, target, slots")
        if ops._held is not None or ops._chain is not None:
            ops.flush_chain()                                # (what waits there may write what is read here)
        ops._on_current(self._table.device)
        n = moves.shape[0]
        rc = self._entry(moves, n, self._table, len(self._tensors), self.pages, self.page_size, self._vector, self._page_bytes, ops._stream())
        if rc in _REFUSED:
            raise KernelError(_REFUSED[rc])
        ops._ok(rc, "copy_pages", -(-n // _MOVES_OF_A_LAUNCH))
