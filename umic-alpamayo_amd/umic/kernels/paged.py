"""Pages of a key / value pool that requests of different lengths share
(libumic_hip.so): block tables and slot maps from request lengths, made on the
device, so that a captured step needs no host in between.

A request's tokens lie in pages of ``page_size`` rows named by its row of
``table``; ``ring`` is the queue of free pages.  ``plan_pages`` makes one step:
tokens dropped, tokens added, pages returned and taken, and for every new token
its slot in the pool and its position.  ``axial.rotate_append`` writes at the
slots; ``attention.cache_attention`` reads through the table.

No counterpart in the reference, whose in-place cache (src/umic/cache.py:25-160)
holds one batch of equal lengths.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from umic import _lib

# status of a step (PageStep.cursor[3])
PLAN_OK, NO_PAGES, TOO_LONG, NO_ROOM, BAD_STATE = range(5)
REFUSALS = {NO_PAGES: "pages are missing", TOO_LONG: "a request is too long",
            NO_ROOM: "too many new tokens", BAD_STATE: "lengths or free pages out of range"}

_I32, _I64 = torch.int32, torch.int64


class PageStep(NamedTuple):
    """What one ``plan_pages`` call gives.

    kv_len:    int32 [R], each request's tokens after the step.
    cursor:    int32 [4], the free queue's head and count, the step's tokens, its
               status (``PLAN_OK`` or why nothing was changed).
    starts:    int32 [R + 1], running sums of the new lengths.
    slots:     int64 [tokens], each new token's row in the pool, -1 where there is none.
    positions: int64 [tokens], its position (plus ``delta``), 0 where there is none.
    """

    kv_len: torch.Tensor
    cursor: torch.Tensor
    starts: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor


def page_size_ok(page_size: int) -> bool:
    """Page sizes the kernels take: powers of two from 16."""
    return page_size >= 16 and page_size & (page_size - 1) == 0


def _refuse(name: str, t: torch.Tensor, n: int, dtype: torch.dtype) -> None:
    raise ValueError(f"plan_pages: {name} must be a contiguous {dtype} vector of {n} on kv_len's "
                     f"device, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _vector(name: str, t: torch.Tensor, n: int, dtype: torch.dtype, dev: int) -> None:
    if (t.dtype is not dtype or t.shape != (n,) or t.get_device() != dev
            or not t.is_contiguous()):
        _refuse(name, t, n, dtype)


def plan_pages(kv_len: torch.Tensor, new_len: torch.Tensor, table: torch.Tensor,
               ring: torch.Tensor, cursor: torch.Tensor, page_size: int, tokens: int, *,
               keep: torch.Tensor | None = None, delta: torch.Tensor | None = None,
               row: int = 0, out: PageStep | None = None) -> PageStep:
    """One step of a paged pool (umic_page_plan).

    Args:
        kv_len: int32 [R], tokens each request holds.
        new_len: int32 [R], tokens it gets.
        table: int32 [R, W], its pages in order; changed entries are written in place.
        ring: int32 [pages], the queue of free pages, written in place.
        cursor: int32 [4], the queue's head and count (the rest is not read).
        page_size: rows of a page, a power of two from 16.
        tokens: entries of slots and positions, at least the new tokens.
        keep: int32 [R], tokens each request keeps at most (None: all; 0 ends it).
        delta: int32 [R], added to each request's positions.
        row: 0, new tokens one request after the other; else request r's begin at
            entry r * row, and tokens is R * row.
        out: where the results go; its kv_len and cursor may be the inputs.

    A step that cannot be made (``cursor[3]`` of the result) changes nothing.
    """
    if not kv_len.is_cuda:
        raise ValueError(f"umic kernels run on the GPU; got a tensor on {kv_len.device}")
    dev, R = kv_len.get_device(), kv_len.shape[0] if kv_len.dim() == 1 else -1
    _vector("kv_len", kv_len, R, _I32, dev)
    _vector("new_len", new_len, R, _I32, dev)
    pages = ring.shape[0] if ring.dim() == 1 else -1
    _vector("ring", ring, pages, _I32, dev)
    _vector("cursor", cursor, 4, _I32, dev)
    if keep is not None:
        _vector("keep", keep, R, _I32, dev)
    if delta is not None:
        _vector("delta", delta, R, _I32, dev)
    if (table.dtype is not _I32 or table.dim() != 2 or table.shape[0] != R
            or table.stride(1) != 1 or table.get_device() != dev):
        raise ValueError(f"plan_pages: table must be int32 [{R}, W] with contiguous rows on "
                         f"kv_len's device, got {table.dtype} {tuple(table.shape)}")
    if not page_size_ok(page_size):
        raise ValueError(f"plan_pages: page_size {page_size} is not a power of two from 16")
    if tokens < 0 or row < 0 or (row and tokens != R * row):
        raise ValueError(f"plan_pages: {tokens} entries for {R} requests of {row} each")
    _lib.lib()
    if out is None:
        ints = torch.empty(2 * R + 5, dtype=_I32, device=kv_len.device)
        longs = torch.empty(2, tokens, dtype=_I64, device=kv_len.device)
        out = PageStep(*ints.split_with_sizes((R, 4, R + 1)), *longs.unbind())
    else:
        for name, n, dtype in (("kv_len", R, _I32), ("cursor", 4, _I32), ("starts", R + 1, _I32),
                               ("slots", tokens, _I64), ("positions", tokens, _I64)):
            _vector("out." + name, getattr(out, name), n, dtype, dev)
    if R == 0:
        out.cursor.copy_(cursor)
        out.cursor[2:] = 0
        out.starts.zero_()
        out.slots.fill_(-1)
        out.positions.zero_()
        return out
    with _lib.device_of(kv_len):
        _lib.call("umic_page_plan", kv_len.data_ptr(), new_len.data_ptr(), _lib.ptr(keep),
                  _lib.ptr(delta), table.data_ptr(), ring.data_ptr(), cursor.data_ptr(),
                  out.kv_len.data_ptr(), out.cursor.data_ptr(), out.starts.data_ptr(),
                  out.slots.data_ptr(), out.positions.data_ptr(), R, table.shape[1],
                  table.stride(0) if R > 1 else table.shape[1], pages, page_size, tokens,
                  row, _lib.stream_of(kv_len))
    return out
