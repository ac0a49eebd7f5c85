"""Attention of new tokens over a key / value cache on gfx950 (libumic_hip.so):
the decode step's single tokens, an action expert's few, a prompt's next chunk.

The cache is contiguous (``umic.cache.KVArena``'s layer views) or paged
(``paged.plan_pages``); it is read where it lies, once, by workgroups that share
the keys of all requests evenly, and their parts are joined.  In the reference the
cache hands such steps to the library's attention, single tokens as a copy of the
whole prefix (src/umic/cache.py:50-80).

Numerics: bf16 products in fp32, softmax in fp32, one rounding of the output.
"""

from __future__ import annotations

import functools

import torch

from umic import _lib
from umic.kernels._common import grad_needed, require_device

HEAD_DIMS = (64, 128, 256)
_BF16 = torch.bfloat16


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(dev: int, S: int, Hq: int, Hk: int, D: int) -> int:
    return _lib.lib().umic_cache_attention_workspace_bytes(S, Hq, Hk, D)


@functools.lru_cache(maxsize=1024)
def max_requests(S: int, Hq: int, Hk: int, D: int, cap: int) -> int:
    """Requests of S new tokens and up to cap keys that one launch takes; 0: not even one."""
    return _lib.lib().umic_cache_attention_max_requests(S, Hq, Hk, D, cap)


# Asked at every call: without the public function's own look at the build.
_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing",
                     None) or torch.cuda.is_current_stream_capturing

# (counters, workspace) of each (device, stream): calls on one stream do not
# overlap, and every call leaves the counters at zero.  A captured call has a
# workspace of its own and no counters, as its graph may run beside anything.
# The latest SCRATCH_STREAMS are held (68 MB each for more than 64 rows of 128);
# what goes was allocated on its stream, and waits for it before it is used again.
SCRATCH_STREAMS = 4
_SCRATCH: dict[tuple[int, int], tuple[torch.Tensor, torch.Tensor]] = {}


def _scratch(q: torch.Tensor, dev: int, stream: int, need: int) -> tuple[int | None, torch.Tensor]:
    if _capturing():
        return None, torch.empty(need, dtype=torch.uint8, device=q.device)
    held = _SCRATCH.get((dev, stream))
    if held is None or held[1].numel() < need:
        counters = held[0] if held else torch.zeros(_lib.UMIC_ATTENTION_COUNTERS,
                                                    dtype=torch.int32, device=q.device)
        held = counters, torch.empty(need, dtype=torch.uint8, device=q.device)
        for key in [] if (dev, stream) in _SCRATCH else list(_SCRATCH)[:1 - SCRATCH_STREAMS]:
            _SCRATCH.pop(key, None)
        _SCRATCH[dev, stream] = held
    return held[0].data_ptr(), held[1]


def _chunks_ok(t: torch.Tensor) -> bool:
    """Contiguous rows of 16-byte chunks."""
    a, b, c, inner = t.stride()
    return inner == 1 and not ((a | b | c) & 7 or t.data_ptr() & 15)


def cache_ok(k_cache: torch.Tensor, v_cache: torch.Tensor) -> bool:
    """Caches the kernel reads: bf16 GPU [blocks, Hk, rows, D] of one layout, D one of
    HEAD_DIMS, 16-byte chunks."""
    return (k_cache.is_cuda and k_cache.dtype is _BF16 and v_cache.dtype is _BF16
            and v_cache.get_device() == k_cache.get_device() and k_cache.dim() == 4
            and _layout_ok(k_cache, v_cache))


def _layout_ok(k_cache: torch.Tensor, v_cache: torch.Tensor) -> bool:
    shape = k_cache.shape
    return (shape == v_cache.shape and shape[3] in HEAD_DIMS
            and k_cache.stride() == v_cache.stride() and v_cache.data_ptr() & 15 == 0
            and _chunks_ok(k_cache))


def _lengths(name: str, t: torch.Tensor, B: int, dev: int) -> None:
    if (t.dtype is not torch.int32 or t.dim() != 1 or t.shape[0] != B or t.get_device() != dev
            or not t.is_contiguous()):
        raise ValueError(f"cache_attention: {name} must be a contiguous int32 vector of {B} on "
                         f"q's device, got {t.dtype} {tuple(t.shape)} on {t.device}")


def cache_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, kv_len, *,
                    table: torch.Tensor | None = None, q_len: torch.Tensor | None = None,
                    causal: bool = True, scale: float | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale q k^T) v of the last S tokens of each request over its cache.

    Args:
        q: [B, Hq, S, D], rotated queries of the new tokens.
        k_cache, v_cache: [B, Hk, rows, D] (request b's rows in block b), or with
            ``table`` [pages, Hk, page_size, D].  The new tokens' rows are in them.
        kv_len: tokens of each request, the new ones included: an int for all, or int32
            [B] on the device (clamped there to what the cache can hold).
        table: int32 [B, W], request b's pages in order.  page_size: a power of two from 16.
        q_len: int32 [B], new tokens of each request (None: S); rows past it are zero.
        causal: new token s sees keys up to its own, kv_len - q_len + s; else all.
        scale: of the scores (None: D ** -0.5).
        out: [B, S, Hq, D] to write to.

    Returns [B, S, Hq, D].  A row that sees no key is zero.
    """
    require_device(q, k_cache, v_cache)
    if grad_needed(q, k_cache, v_cache):
        raise RuntimeError("cache_attention: the kernel has no backward; call it under "
                           "torch.no_grad()")
    shape, cshape = q.shape, k_cache.shape
    if len(shape) != 4 or len(cshape) != 4 or not _layout_ok(k_cache, v_cache):
        raise ValueError(f"cache_attention: unsupported layout q{tuple(shape)} "
                         f"cache{tuple(cshape)} (head sizes {HEAD_DIMS})")
    B, Hq, S, D = shape
    blocks, Hk, rows, Dk = cshape
    if Dk != D or Hk == 0 or Hq % Hk:
        raise ValueError(f"cache_attention: {Hq} heads of {D} over a cache of {Hk} of {Dk}")
    dev = q.get_device()
    if table is None:
        if blocks != B:
            raise ValueError(f"cache_attention: {B} requests over a cache of {blocks} blocks")
        cap, ld, width = rows, 0, 0
    else:
        if (table.dtype is not torch.int32 or table.dim() != 2 or table.shape[0] != B
                or table.shape[1] == 0 or table.get_device() != dev or table.stride(1) != 1):
            raise ValueError(f"cache_attention: table must be int32 [{B}, W > 0] with contiguous "
                             f"rows on q's device, got {table.dtype} {tuple(table.shape)}")
        width = table.shape[1]
        cap, ld = width * rows, table.stride(0) if B > 1 else width
    if isinstance(kv_len, torch.Tensor):
        _lengths("kv_len", kv_len, B, dev)
        lens, n = kv_len.data_ptr(), 0
    else:
        lens, n = None, int(kv_len)
        if not 0 <= n <= cap:
            raise ValueError(f"cache_attention: kv_len {n} of a cache that holds {cap}")
    if q_len is not None:
        _lengths("q_len", q_len, B, dev)
    if not _chunks_ok(q):
        q = q.clone(memory_format=torch.contiguous_format)
    if out is None:
        out = torch.empty(B, S, Hq, D, dtype=_BF16, device=q.device)
        os_ = (S * Hq * D, Hq * D, D)
    else:
        require_device(q, out)
        if tuple(out.shape) != (B, S, Hq, D) or not _chunks_ok(out):
            raise ValueError(f"cache_attention: out must be [{B}, {S}, {Hq}, {D}] of 16-byte "
                             f"chunks, got {tuple(out.shape)}")
        os_ = out.stride()
        if any(st == 0 and n > 1 for st, n in zip(os_, out.shape)):
            raise ValueError("cache_attention: out must not share rows")
    if B == 0 or S == 0 or Hq == 0:
        return out
    most = max_requests(S, Hq, Hk, D, cap)
    if B > most:
        if most == 0:
            raise ValueError(f"cache_attention: {S} new tokens of {Hq} heads over up to {cap} keys "
                             "are too many for one launch")
        for b in range(0, B, most):  # requests stand for themselves
            part = slice(b, b + most)
            kv = (k_cache, v_cache) if table is not None else (k_cache[part], v_cache[part])
            cache_attention(q[part], *kv, n if lens is None else kv_len[part],
                            table=None if table is None else table[part],
                            q_len=None if q_len is None else q_len[part], causal=causal,
                            scale=scale, out=out[part])
        return out
    qs, cs = q.stride(), k_cache.stride()
    with _lib.device_of(q):
        stream = _lib.stream_of(q)
        size = _workspace_bytes(dev, S, Hq, Hk, D)
        counters, ws = _scratch(q, dev, stream, size)
        _lib.call("umic_cache_attention_bf16", q.data_ptr(), k_cache.data_ptr(),
                  v_cache.data_ptr(), out.data_ptr(), _lib.ptr(table), lens, _lib.ptr(q_len),
                  B, S, Hq, Hk, D, qs[0], qs[2], qs[1], os_[0], os_[1], os_[2], cs[0], cs[1],
                  cs[2], blocks, rows, ld, width, n, int(causal),
                  float(D ** -0.5 if scale is None else scale), counters,
                  ws.data_ptr(), size, stream)
    return out
