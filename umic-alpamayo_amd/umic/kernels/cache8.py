"""A paged key / value cache in 8 bits on gfx950 (libumic_hip.so): twice the tokens of a
pool, and half the bytes of a decode step (over 260000 keys in all half the time, over 25000
two thirds, over one prompt's 3100 the same).

``Pages8`` holds codes, ``torch.int8`` or ``torch.float8_e4m3fn``, and a scale for each
block of ``BLOCK`` = 16 consecutive rows of a page, of one key head.  Scales are powers of
two, so that a code times its scale is a bf16 number (at the top of its range the largest
one): what ``read`` gives is what ``attention`` sees.  Requests, tables, slots and lengths
are ``paged.plan_pages``'s.

Writing.  ``rotate_append`` is ``axial.rotate_append`` with the rows quantised, and
``append`` writes k as it comes.  A block's scale follows the largest magnitude a among
the rows that come into it: 2^(floor(log2 a) - 6) for int8 (the largest code is 64 to
127), - 7 for e4m3, 2^-100 at least.  Where the block holds tokens already (the lowest
row that comes is not its first) it stays at least what it was, and where it grows, the
rows before are rounded to it; its other rows count as dropped.  An
int8 value is off by half a scale at most as it is written, and by one scale at most
after its block's scale has grown; an e4m3 value of 2^-6 scales and more by 2^-4 of
itself.  A NaN or an infinity makes its block's scale NaN until the block is begun anew:
all of it reads as NaN, tokens written before too, also after that token is dropped.

No counterpart in the reference, whose cache (src/umic/cache.py:25-160) is of 16-bit rows.
"""

from __future__ import annotations

import ctypes
import functools
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


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(dev: int, S: int, Hq: int, Hk: int, D: int) -> int:
    return _lib.lib().umic_cache8_attention_workspace_bytes(S, Hq, Hk, D)


class _Layout(NamedTuple):
    """What the kernels are told of a cache, and where it was looked at."""

    pointers: tuple
    struct: _lib.Cache8
    at: int  # the structure's address
    pages: int
    heads: int
    page_size: int
    head_dim: int
    apart: bool  # no two rows or scales share memory


class _Fields(NamedTuple):
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


class Pages8(_Fields):
    """k, v: codes [pages, Hk, page_size, D] of one type and layout, rows of 16-byte
    chunks; k_scale, v_scale: fp32 [pages, Hk, page_size / BLOCK], powers of two.  Looked at
    at its first use, and again where its tensors have moved: one object for many calls saves
    looking.  Their shapes and strides are not changed in place (``transpose_``,
    ``resize_``), nor are they made to require a gradient.  Rows or scales that share memory
    (``expand``) can be read, not written."""

    def __reduce__(self):  # copies look for themselves
        return type(self), tuple(self)

    def layout(self, who: str, dev: int) -> _Layout:
        """Its layout on device dev; raises where the kernels do not take it."""
        held = self.__dict__.get("_held")
        k, v, ks, vs = self
        if (held is not None and held[0] == dev and held[1].pointers
                == (k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr())):
            return held[1]
        got = _look(who, self, dev)
        self._held = dev, got
        return got


def empty(pages: int, heads: int, page_size: int, head_dim: int,
          dtype: torch.dtype = torch.int8, device: torch.device | str = "cuda") -> Pages8:
    """Pages that hold nothing yet."""
    if dtype not in DTYPES or head_dim not in HEAD_DIMS or not paged.page_size_ok(page_size):
        raise ValueError(f"cache8.empty: {dtype} (one of {list(DTYPES)}), head_dim {head_dim} (one "
                         f"of {HEAD_DIMS}), page_size {page_size} (powers of two from 16)")
    k, v = torch.empty(2, pages, heads, page_size, head_dim, dtype=dtype, device=device)
    k_scale, v_scale = torch.ones(2, pages, heads, page_size // BLOCK, device=device)
    return Pages8(k, v, k_scale, v_scale)


def _apart(shape, strides, width: int, between: int) -> bool:
    """Whether blocks of ``width`` bytes, at these strides in bytes, lie each for itself (the
    strides nest), and those of a second tensor of the layout ``between`` bytes on between
    them."""
    dims, span = [], width
    for st, n in sorted((st, n) for st, n in zip(strides, shape) if n > 1):
        if st < span:
            return False
        dims.append((st, n))
        span += st * (n - 1)

    def meet(gap: int, inner: int) -> bool:
        if inner == 0:
            return abs(gap) < width
        st, n = dims[inner - 1]
        return any(abs(m) < n and meet(gap - m * st, inner - 1) for m in (gap // st, gap // st + 1))

    return 0 in shape or not meet(between, len(dims))


def _look(who: str, cache: Pages8, dev: int) -> _Layout:
    k, v, ks, vs = cache
    shape, st, sst = k.shape, k.stride(), ks.stride()
    if (k.dtype not in DTYPES or v.dtype is not k.dtype or len(shape) != 4 or shape != v.shape
            or shape[3] not in HEAD_DIMS or shape[1] == 0 or st != v.stride() or st[3] != 1
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
    if any(t.requires_grad for t in cache):
        raise RuntimeError(f"{who}: the cache has no gradient; its tensors must not require one")
    pointers = tuple(t.data_ptr() for t in cache)
    struct = _lib.Cache8(*pointers, shape[0], shape[2], shape[1], shape[3], st[0], st[1], st[2],
                         sst[0], sst[1], DTYPES[k.dtype])
    apart = (_apart(shape[:3], st[:3], shape[3], pointers[1] - pointers[0])
             and _apart(ks.shape, [4 * n for n in sst], 4, pointers[3] - pointers[2]))
    return _Layout(pointers, struct, ctypes.addressof(struct), *shape, apart)


def _chunks16(t: torch.Tensor) -> tuple[torch.Tensor, int, int]:
    """t [T, H, D], or a copy, with rows of 16-byte chunks; and its strides."""
    a, b, inner = t.stride()
    if inner == 1 and not ((a | b) & 7 or t.data_ptr() & 15):
        return t, a, b
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.stride(0), t.stride(1)


def _rows(who: str, k, v, slots, cache: Pages8) -> tuple[_Layout, tuple, tuple]:
    """The checks and row views that both appends share."""
    shape, dev = k.shape, k.get_device()
    lay = cache.layout(who, dev)
    if len(shape) != 3 or v.shape != shape or shape[1] != lay.heads or shape[2] != lay.head_dim:
        raise ValueError(f"{who}: k {tuple(shape)} and v {tuple(v.shape)} must be [T, {lay.heads}, "
                         f"{lay.head_dim}], as the pages")
    if not lay.apart:
        raise ValueError(f"{who}: rows or scales of the cache share memory")
    if (slots.dtype is not torch.int64 or slots.shape != shape[:1] or slots.get_device() != dev
            or not slots.is_contiguous()):
        raise ValueError(f"{who}: slots must be a contiguous int64 vector of {shape[0]} on k's device")
    return lay, _chunks16(k), _chunks16(v)


def rotate_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                  plan: axial.AxisPlan, slots: torch.Tensor, cache: Pages8,
                  norm=None) -> torch.Tensor:
    """``axial.rotate`` of q and k (norm: ``(q_w, k_w, eps)``), their angles rounded finer
    than there (within a quarter turn; not its bits), k's rotated rows and v's rows written
    as codes to ``slots`` (int64 [T], distinct, in any order; one outside the pool writes
    nothing).  Quickest where a block's tokens (slots that differ below BLOCK
    only) stand within 24 neighbouring ones, as ``paged.plan_pages`` has them.  Returns the
    rotated q."""
    require_device(q, k, v, *(norm[:2] if norm is not None else ()))
    axial._check("cache8.rotate_append", q, k, positions, plan, norm)
    if grad_needed(v):
        raise RuntimeError("cache8.rotate_append: the kernel has no backward; call it under "
                           "torch.no_grad()")
    lay, (k, k0, k1), (v, v0, v1) = _rows("cache8.rotate_append", k, v, slots, cache)
    q, q0, q1 = _chunks16(q)
    T, Hq, D = q.shape
    qw, kw, eps = axial._norm_args("cache8.rotate_append", norm, D)
    if norm is not None and (qw | kw) & 15:
        raise ValueError("cache8.rotate_append: norm weights must be 16-byte aligned")
    out = q.new_empty((T, Hq, D))
    p0, p1 = positions.stride()
    with _lib.device_of(q):
        _lib.call("umic_cache8_append_bf16", lay.at, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                  out.data_ptr(), positions.data_ptr(), plan.turn.data_ptr(), plan.axis.data_ptr(),
                  slots.data_ptr(), plan.scale, qw, kw, eps, T, Hq, positions.shape[0], p0, p1, q0,
                  q1, k0, k1, v0, v1, _lib.stream_of(q))
    return out


def append(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, cache: Pages8) -> None:
    """Rows of k and v [T, heads, D] written as codes to ``slots``, as ``rotate_append``
    does, without a rotation."""
    require_device(k, v)
    if grad_needed(k, v):
        raise RuntimeError("cache8.append: the kernel has no backward; call it under "
                           "torch.no_grad()")
    lay, (k, k0, k1), (v, v0, v1) = _rows("cache8.append", k, v, slots, cache)
    with _lib.device_of(k):
        _lib.call("umic_cache8_append_bf16", lay.at, None, k.data_ptr(), v.data_ptr(), None, None,
                  None, None, slots.data_ptr(), 1.0, None, None, 0.0, k.shape[0], 0, 0, 0, 0, 0, 0,
                  k0, k1, v0, v1, _lib.stream_of(k))


def _requests(who: str, table: torch.Tensor, kv_len, page_size: int, dev: int) -> tuple:
    """(B, table width, its row stride, lengths' pointer, length of all)."""
    shape, st = table.shape, table.stride()
    if (table.dtype is not torch.int32 or len(shape) != 2 or shape[1] == 0
            or table.get_device() != dev or st[1] != 1 and shape[1] > 1):
        raise ValueError(f"{who}: table must be int32 [requests, W > 0] with contiguous rows on the "
                         f"cache's device, got {table.dtype} {tuple(table.shape)}")
    B, width = shape
    ld = st[0] if B > 1 else width
    if isinstance(kv_len, torch.Tensor):
        _bf16._lengths("kv_len", kv_len, B, dev)
        return B, width, ld, kv_len.data_ptr(), 0
    n = int(kv_len)
    if not 0 <= n <= width * page_size:
        raise ValueError(f"{who}: kv_len {n} of a table that holds {width * page_size}")
    return B, width, ld, None, n


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
    dev = table.get_device()
    if dev < 0:
        raise ValueError(f"umic kernels run on the GPU; got a tensor on {table.device}")
    lay = cache.layout("cache8.read", dev)
    B, width, ld, lens, n = _requests("cache8.read", table, kv_len, lay.page_size, dev)
    if rows < 0:
        raise ValueError(f"cache8.read: {rows} rows")
    if start is not None:
        _bf16._lengths("start", start, B, dev)
    shape = (B, lay.heads, rows, lay.head_dim)
    k = table.new_empty(shape, dtype=_BF16)
    v = torch.empty_like(k)
    with _lib.device_of(k):
        _lib.call("umic_cache8_read_bf16", lay.at, k.data_ptr(), v.data_ptr(), table.data_ptr(),
                  lens, _lib.ptr(start), B, rows, ld, width, n, _lib.stream_of(k))
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
    dev, shape = q.get_device(), q.shape
    lay = cache.layout("cache8.attention", dev)
    Hk = lay.heads
    if len(shape) != 4 or shape[3] != lay.head_dim or shape[1] % Hk:
        raise ValueError(f"cache8.attention: q {tuple(shape)} over a cache of {Hk} heads of "
                         f"{lay.head_dim}")
    B, Hq, S, D = shape
    rows, width, ld, lens, n = _requests("cache8.attention", table, kv_len, lay.page_size, dev)
    if rows != B:
        raise ValueError(f"cache8.attention: {B} requests over a table of {rows}")
    if q_len is not None:
        _bf16._lengths("q_len", q_len, B, dev)
    if not _bf16._chunks_ok(q):
        q = q.clone(memory_format=torch.contiguous_format)
    if out is None:
        out = q.new_empty((B, S, Hq, D))
        o0, o1, o2 = S * Hq * D, Hq * D, D
    else:
        require_device(q, out)
        if tuple(out.shape) != (B, S, Hq, D) or not _bf16._chunks_ok(out):
            raise ValueError(f"cache8.attention: out must be [{B}, {S}, {Hq}, {D}] of 16-byte "
                             f"chunks, got {tuple(out.shape)}")
        if any(st == 0 and m > 1 for st, m in zip(out.stride(), out.shape)):
            raise ValueError("cache8.attention: out must not share rows")
        o0, o1, o2, _ = out.stride()
    if B == 0 or S == 0 or Hq == 0:
        return out
    most = _bf16.max_requests(S, Hq, Hk, D, width * lay.page_size)
    if B > most:
        if most == 0:
            raise ValueError(f"cache8.attention: {S} new tokens of {Hq} heads over up to "
                             f"{width * lay.page_size} keys are too many for one launch")
        for b in range(0, B, most):  # requests stand for themselves
            part = slice(b, b + most)
            attention(q[part], cache, n if lens is None else kv_len[part], table[part],
                      q_len=None if q_len is None else q_len[part], causal=causal, scale=scale,
                      out=out[part])
        return out
    q0, q1, q2, _ = q.stride()
    with _lib.device_of(q):
        stream = _lib.stream_of(q)
        size = _workspace_bytes(dev, S, Hq, Hk, D)
        counters, ws = _bf16._scratch(q, dev, stream, size)
        _lib.call("umic_cache8_attention_bf16", lay.at, q.data_ptr(), out.data_ptr(),
                  table.data_ptr(), lens, _lib.ptr(q_len), B, S, Hq, q0, q2, q1, o0, o1, o2, ld,
                  width, n, int(causal), float(D ** -0.5 if scale is None else scale), counters,
                  ws.data_ptr(), size, stream)
    return out
