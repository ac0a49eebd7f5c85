"""A paged key / value cache in 8 bits on gfx950 (libumic_hip.so): half the bytes of a
decode step, twice the tokens of a pool.

``Pages8`` holds codes, ``torch.int8`` or ``torch.float8_e4m3fn``, and a scale for each
block of ``BLOCK`` = 16 consecutive rows of a page, of one key head.  Scales are powers of
two, so that a code times its scale is a bf16 number: what ``read`` gives is what
``attention`` sees.  Requests, tables, slots and lengths are ``paged.plan_pages``'s.

Writing.  ``rotate_append`` is ``axial.rotate_append`` with the rows quantised, and
``append`` writes k as it comes.  A block's scale follows the largest magnitude a among
the rows that come into it: 2^(floor(log2 a) - 6) for int8 (the largest code is 64 to
127), - 7 for e4m3, 2^-100 at least.  Where the block holds tokens already (the lowest
row that comes is not its first) it stays at least what it was, and where it grows, the
rows before are rounded to it; its other rows count as dropped.  An
int8 value is off by half a scale at most as it is written, and by one scale at most
after its block's scale has grown; an e4m3 value of 2^-6 scales and more by 2^-4 of
itself.  A NaN or an infinity makes its block's scale NaN until the block is begun anew:
all of it reads as NaN.

No counterpart in the reference, whose cache (src/umic/cache.py:25-160) is of 16-bit rows.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from umic import _lib
from umic.kernels import attention as _bf16
from umic.kernels import axial, paged
from umic.kernels._common import grad_needed, require_device

BLOCK = 16  # rows that share a scale
DTYPES = {torch.float8_e4m3fn: _lib.UMIC_CODES_E4M3, torch.int8: _lib.UMIC_CODES_INT8}
HEAD_DIMS = _bf16.HEAD_DIMS
_BF16 = torch.bfloat16


class Pages8(NamedTuple):
    """k, v: codes [pages, Hk, page_size, D] of one type and layout, rows of 16-byte
    chunks; k_scale, v_scale: fp32 [pages, Hk, page_size / BLOCK], powers of two."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


def empty(pages: int, heads: int, page_size: int, head_dim: int,
          dtype: torch.dtype = torch.int8, device: torch.device | str = "cuda") -> Pages8:
    """Pages that hold nothing yet."""
    if dtype not in DTYPES or head_dim not in HEAD_DIMS or not paged.page_size_ok(page_size):
        raise ValueError(f"cache8.empty: {dtype} (one of {list(DTYPES)}), head_dim {head_dim} (one "
                         f"of {HEAD_DIMS}), page_size {page_size} (powers of two from 16)")
    k, v = torch.empty(2, pages, heads, page_size, head_dim, dtype=dtype, device=device)
    k_scale, v_scale = torch.ones(2, pages, heads, page_size // BLOCK, device=device)
    return Pages8(k, v, k_scale, v_scale)


def _pages(who: str, cache: Pages8, dev: int) -> tuple:
    """(format, shape, code strides, scale strides) of a cache on device dev."""
    k, v, ks, vs = cache
    shape, st, sst = k.shape, k.stride(), ks.stride()
    if (k.dtype not in DTYPES or v.dtype is not k.dtype or len(shape) != 4 or shape != v.shape
            or shape[3] not in HEAD_DIMS or st != v.stride() or st[3] != 1
            or (st[0] | st[1] | st[2] | k.data_ptr() | v.data_ptr()) & 15):
        raise ValueError(f"{who}: codes k {k.dtype} {tuple(shape)} and v {v.dtype} {tuple(v.shape)} "
                         f"must be of one type ({list(DTYPES)}) and layout, [pages, heads, "
                         f"page_size, D (one of {HEAD_DIMS})] in chunks of 16 bytes")
    if (not paged.page_size_ok(shape[2]) or ks.dtype is not torch.float32
            or vs.dtype is not torch.float32 or ks.shape != (*shape[:2], shape[2] // BLOCK)
            or vs.shape != ks.shape or sst != vs.stride() or sst[2] != 1 and ks.shape[2] > 1):
        raise ValueError(f"{who}: scales must be fp32 [pages, heads, page_size / {BLOCK}] of one "
                         f"layout (page_size a power of two from 16), got {ks.dtype} "
                         f"{tuple(ks.shape)} and {vs.dtype} {tuple(vs.shape)} for pages {tuple(shape)}")
    if any(t.get_device() != dev for t in cache):
        raise ValueError(f"{who}: the cache is on {k.device}, not with the other tensors")
    return DTYPES[k.dtype], shape, st, sst


def _chunks16(t: torch.Tensor) -> torch.Tensor:
    """t [T, H, D], or a copy, with rows of 16-byte chunks."""
    a, b, inner = t.stride()
    if inner == 1 and not ((a | b) & 7 or t.data_ptr() & 15):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _store(who: str, q, k, v, positions, plan, slots, cache: Pages8, norm):
    """The append of ``rotate_append`` and, q None, of ``append``."""
    shape = k.shape
    if len(shape) != 3 or v.shape != shape or shape[1] == 0:
        raise ValueError(f"{who}: k {tuple(shape)} and v {tuple(v.shape)} must be [T, heads, D]")
    T, Hk, D = shape
    fmt, pages, cst, sst = _pages(who, cache, k.get_device())
    if pages[1] != Hk or pages[3] != D:
        raise ValueError(f"{who}: {Hk} heads of {D} into pages of {pages[1]} of {pages[3]}")
    if (slots.dtype is not torch.int64 or slots.shape != (T,)
            or slots.get_device() != k.get_device() or not slots.is_contiguous()):
        raise ValueError(f"{who}: slots must be a contiguous int64 vector of {T} on k's device")
    k, v = _chunks16(k), _chunks16(v)
    if q is None:
        out, turns, heads = None, (None, None, None, None), (None, None, 0.0)
        Hq, axes, ps, qs, os_, scale = 0, 0, (0, 0), (0, 0), (0, 0), 1.0
    else:
        q, Hq = _chunks16(q), q.shape[1]
        out = torch.empty(T, Hq, D, dtype=_BF16, device=q.device)
        turns = (positions.data_ptr(), plan.turn.data_ptr(), plan.axis.data_ptr())
        heads = axial._norm_args(who, norm, D)
        if norm is not None and (norm[0].data_ptr() | norm[1].data_ptr()) & 15:
            raise ValueError(f"{who}: norm weights must be 16-byte aligned")
        axes, ps, qs, os_, scale = (positions.shape[0], positions.stride(), q.stride(),
                                    (Hq * D, D), plan.scale)
    with _lib.device_of(k):
        _lib.call("umic_cache8_append_bf16", _lib.ptr(q), k.data_ptr(), v.data_ptr(),
                  _lib.ptr(out), *(t.data_ptr() for t in cache), *turns[:3], slots.data_ptr(),
                  scale, *heads, T, Hq, Hk, D, axes, ps[0], ps[1], qs[0], qs[1], k.stride(0),
                  k.stride(1), v.stride(0), v.stride(1), *os_, cst[0], cst[1], cst[2], sst[0],
                  sst[1], pages[0], pages[2], fmt, _lib.stream_of(k))
    return out


def rotate_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                  plan: axial.AxisPlan, slots: torch.Tensor, cache: Pages8,
                  norm=None) -> torch.Tensor:
    """``axial.rotate`` of q and k (norm: ``(q_w, k_w, eps)``), k's rotated rows and v's
    rows written as codes to ``slots`` (int64 [T], distinct; one outside the pool writes
    nothing).  The tokens of one block (slots that differ below BLOCK only) stand within 24
    neighbouring tokens, as ``paged.plan_pages`` has them next to each other.  Returns the
    rotated q."""
    require_device(q, k, v, *(norm[:2] if norm is not None else ()))
    axial._check("cache8.rotate_append", q, k, positions, plan, norm)
    if grad_needed(v):
        raise RuntimeError("cache8.rotate_append: the kernel has no backward; call it under "
                           "torch.no_grad()")
    return _store("cache8.rotate_append", q, k, v, positions, plan, slots, cache, norm)


def append(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, cache: Pages8) -> None:
    """Rows of k and v [T, heads, D] written as codes to ``slots``, as ``rotate_append``
    does, without a rotation."""
    require_device(k, v)
    if grad_needed(k, v):
        raise RuntimeError("cache8.append: the kernel has no backward; call it under "
                           "torch.no_grad()")
    _store("cache8.append", None, k, v, None, None, slots, cache, None)


def _requests(who: str, table: torch.Tensor, kv_len, page_size: int, dev: int) -> tuple:
    """(B, table width, its row stride, lengths' pointer, length of all)."""
    if (table.dtype is not torch.int32 or table.dim() != 2 or table.shape[1] == 0
            or table.get_device() != dev or table.stride(1) != 1 and table.shape[1] > 1):
        raise ValueError(f"{who}: table must be int32 [requests, W > 0] with contiguous rows on the "
                         f"cache's device, got {table.dtype} {tuple(table.shape)}")
    B, width = table.shape
    if isinstance(kv_len, torch.Tensor):
        _bf16._lengths("kv_len", kv_len, B, dev)
        return B, width, table.stride(0) if B > 1 else width, kv_len.data_ptr(), 0
    n = int(kv_len)
    if not 0 <= n <= width * page_size:
        raise ValueError(f"{who}: kv_len {n} of a table that holds {width * page_size}")
    return B, width, table.stride(0) if B > 1 else width, None, n


def read(cache: Pages8, table: torch.Tensor, kv_len, rows: int, *,
         start: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values as bf16, exactly: two [B, Hk, rows, D], row i of request b being its
    token start[b] + i.

    Args:
        table: int32 [B, W], request b's pages in order.
        kv_len: tokens of each request, an int for all or int32 [B]; rows past it are zero.
        rows: rows to read of each request.
        start: int32 [B], the first one (None: 0).
    """
    dev = cache.k.get_device()
    if dev < 0:
        raise ValueError(f"umic kernels run on the GPU; got a tensor on {cache.k.device}")
    fmt, shape, cst, sst = _pages("cache8.read", cache, dev)
    B, width, ld, lens, n = _requests("cache8.read", table, kv_len, shape[2], dev)
    if rows < 0:
        raise ValueError(f"cache8.read: {rows} rows")
    if start is not None:
        _bf16._lengths("start", start, B, dev)
    _lib.lib()
    k, v = torch.empty(2, B, shape[1], rows, shape[3], dtype=_BF16, device=cache.k.device)
    with _lib.device_of(k):
        _lib.call("umic_cache8_read_bf16", *(t.data_ptr() for t in cache), k.data_ptr(),
                  v.data_ptr(), table.data_ptr(), lens, _lib.ptr(start), B, shape[1], rows,
                  shape[3], cst[0], cst[1], cst[2], sst[0], sst[1], shape[0], shape[2], ld, width,
                  n, fmt, _lib.stream_of(k))
    return k, v


def attention(q: torch.Tensor, cache: Pages8, kv_len, table: torch.Tensor, *,
              q_len: torch.Tensor | None = None, causal: bool = True,
              scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``attention.cache_attention`` over a cache in 8 bits: softmax(scale q k^T) v of the
    last S tokens of each request, fp32 with one rounding.

    Args:
        q: bf16 [B, Hq, S, D], rotated queries of the new tokens, whose rows are in the cache.
        kv_len: tokens of each request, the new ones included: an int for all, or int32
            [B] on the device (clamped there to what the table can hold).
        table: int32 [B, W], request b's pages in order.
        q_len: int32 [B], new tokens of each request (None: S); rows past it are zero.
        causal: new token s sees keys up to its own, kv_len - q_len + s; else all.
        scale: of the scores (None: D ** -0.5).
        out: [B, S, Hq, D] to write to.

    Returns [B, S, Hq, D].  A row that sees no key is zero.
    """
    require_device(q)
    if grad_needed(q):
        raise RuntimeError("cache8.attention: the kernel has no backward; call it under "
                           "torch.no_grad()")
    dev = q.get_device()
    fmt, shape, cs, sst = _pages("cache8.attention", cache, dev)
    pages, Hk, ps, Dk = shape
    if q.dim() != 4 or q.shape[3] != Dk or Hk == 0 or q.shape[1] % Hk:
        raise ValueError(f"cache8.attention: q {tuple(q.shape)} over a cache of {Hk} heads of {Dk}")
    B, Hq, S, D = q.shape
    rows, width, ld, lens, n = _requests("cache8.attention", table, kv_len, ps, dev)
    if rows != B:
        raise ValueError(f"cache8.attention: {B} requests over a table of {rows}")
    if q_len is not None:
        _bf16._lengths("q_len", q_len, B, dev)
    if not _bf16._chunks_ok(q):
        q = q.clone(memory_format=torch.contiguous_format)
    if out is None:
        out = torch.empty(B, S, Hq, D, dtype=_BF16, device=q.device)
    else:
        require_device(q, out)
        if tuple(out.shape) != (B, S, Hq, D) or not _bf16._chunks_ok(out):
            raise ValueError(f"cache8.attention: out must be [{B}, {S}, {Hq}, {D}] of 16-byte "
                             f"chunks, got {tuple(out.shape)}")
        if any(st == 0 and m > 1 for st, m in zip(out.stride(), out.shape)):
            raise ValueError("cache8.attention: out must not share rows")
    if B == 0 or S == 0 or Hq == 0:
        return out
    most = _bf16.max_requests(S, Hq, Hk, D, width * ps)
    if B > most:
        if most == 0:
            raise ValueError(f"cache8.attention: {S} new tokens of {Hq} heads over up to "
                             f"{width * ps} keys are too many for one launch")
        for b in range(0, B, most):  # requests stand for themselves
            part = slice(b, b + most)
            attention(q[part], cache, n if lens is None else kv_len[part], table[part],
                      q_len=None if q_len is None else q_len[part], causal=causal, scale=scale,
                      out=out[part])
        return out
    qs, os_ = q.stride(), out.stride()
    with _lib.device_of(q):
        stream = _lib.stream_of(q)
        size = _bf16._workspace_bytes(dev, S, Hq, Hk, D)
        counters, ws = _bf16._scratch(q, dev, stream, size)
        _lib.call("umic_cache8_attention_bf16", q.data_ptr(), *(t.data_ptr() for t in cache),
                  out.data_ptr(), table.data_ptr(), lens, _lib.ptr(q_len), B, S, Hq, Hk, D, qs[0],
                  qs[2], qs[1], os_[0], os_[1], os_[2], cs[0], cs[1], cs[2], sst[0], sst[1], pages,
                  ps, ld, width, n, fmt, int(causal),
                  float(D ** -0.5 if scale is None else scale), counters, ws.data_ptr(), size,
                  stream)
    return out
