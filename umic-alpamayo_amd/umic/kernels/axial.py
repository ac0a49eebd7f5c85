"""Rotary embedding from positions of several axes (time, height and width of
images and video) on gfx950 (libumic_hip.so), with the attention's q_norm /
k_norm in front and the append into a paged pool behind, in one launch.

The reference rotates by cos / sin tables that the model makes from the
positions (src/umic/kernels/rope.py:62-107).  Here the positions are the input: an
``AxisPlan`` says which axis turns which pair of a head row, and how fast.

Numerics: fp32 with one rounding to bf16 (the eager text chain rounds the
tables, both products and the sum: ``rope``).  Angles are 64-bit fractions of a
turn, so positions of any size turn exactly.
"""

from __future__ import annotations

from fractions import Fraction

import torch

from umic import _lib
from umic.kernels._common import grad_needed, require_device

MAX_HEAD_DIM = 512
_PI = Fraction(314159265358979323846264338327950288419716939937510582097494, 10 ** 59)
_UNIT = round(2 ** 191 / _PI)  # 2^64 / (2 pi) turns a radian, 128 bits behind the point


def _turn(freq: float) -> int:
    """round(2^64 freq / (2 pi)) modulo 2^64, as a signed number."""
    n, d = freq.as_integer_ratio()
    t = ((n * _UNIT // d >> 127) + 1 >> 1) & 2 ** 64 - 1
    return t - 2 ** 64 if t >= 2 ** 63 else t


class AxisPlan:
    """Which axis turns which pair of a head row, and how fast.

    inv_freq: [D/2] radians per position of each pair (its fp32 values are taken
        exactly); axis: [D/2] the axis whose positions turn it; scale: factor of
        cos and sin (a rotary module's ``attention_scaling``).
    """

    def __init__(self, inv_freq: torch.Tensor, axis, scale: float = 1.0,
                 device: torch.device | str | None = None) -> None:
        device = inv_freq.device if device is None else torch.device(device)
        freq = inv_freq.detach().double().cpu().tolist()
        axis = torch.as_tensor(axis).detach().cpu().to(torch.int32)
        if inv_freq.dim() != 1 or axis.shape != inv_freq.shape:
            raise ValueError(f"AxisPlan: inv_freq {tuple(inv_freq.shape)} and axis "
                             f"{tuple(axis.shape)} must be vectors of one length")
        if not freq or not all(abs(f) < float("inf") for f in freq) or int(axis.min()) < 0:
            raise ValueError("AxisPlan: frequencies must be finite and axes not negative")
        self.turn = torch.tensor([_turn(f) for f in freq], dtype=torch.int64).to(device)
        self.axis = axis.to(device)
        self.axes = int(axis.max()) + 1
        self.head_dim = 2 * len(freq)
        self.scale = float(scale)

    @classmethod
    def text(cls, head_dim: int, theta: float, sections, interleaved: bool = True,
             scale: float = 1.0, device: torch.device | str = "cuda") -> "AxisPlan":
        """The text trunk's plan: pair f turns at theta^(-2 f / head_dim).
        ``sections`` are the pairs of each axis.  Interleaved (Qwen3-VL): axis a >
        0 has pairs a, a + n, a + 2 n .. (n axes), as many as its section, and axis
        0 the rest; else (Qwen2-VL) one axis after the other."""
        half, n = head_dim // 2, len(sections)
        if head_dim % 2 or sum(sections) != half:
            raise ValueError(f"AxisPlan.text: sections {tuple(sections)} are not the {half} pairs "
                             f"of a head of {head_dim}")
        if interleaved:
            axis = [0] * half
            for a in range(1, n):
                for f in range(a, min(half, n * sections[a]), n):
                    axis[f] = a
        else:
            axis = [a for a, s in enumerate(sections) for _ in range(s)]
        inv = 1.0 / theta ** (torch.arange(0, head_dim, 2, dtype=torch.float32) / head_dim)
        return cls(inv, axis, scale, device)

    @classmethod
    def rotary(cls, module: torch.nn.Module) -> "AxisPlan":
        """The plan of a transformers text rotary module: its ``inv_freq``,
        ``mrope_section`` (interleaved) and ``attention_scaling``.  A module that changes
        its frequencies with the longest position it meets is refused."""
        kind = str(getattr(module, "rope_type", "default"))
        if "dynamic" in kind or kind == "longrope":
            raise ValueError(f"AxisPlan.rotary: frequencies of rope type {kind!r} follow the length")
        inv = module.inv_freq
        sections = list(getattr(module, "mrope_section", None) or [inv.shape[0]])
        plan = cls.text(2 * inv.shape[0], 1e4, sections, device="cpu")
        return cls(inv, plan.axis, getattr(module, "attention_scaling", 1.0))

    @classmethod
    def grid(cls, head_dim: int, theta: float = 1e4,
             device: torch.device | str = "cuda") -> "AxisPlan":
        """A vision encoder's plan: the first half of the pairs turns by rows, the
        second by columns, both at theta^(-4 f / head_dim)."""
        if head_dim % 4:
            raise ValueError(f"AxisPlan.grid: a head of {head_dim} has no two halves of pairs")
        half = head_dim // 2
        inv = 1.0 / theta ** (torch.arange(0, half, 2, dtype=torch.float32) / half)
        quarter = half // 2
        return cls(torch.cat((inv, inv)), [0] * quarter + [1] * quarter, device=device)


def _ready(t: torch.Tensor) -> tuple[torch.Tensor, int, int]:
    """t, or a copy with the rows the kernel reads: [T, H, D], contiguous, in 8-byte
    chunks; and its strides."""
    a, b, inner = t.stride()
    if inner == 1 and not ((a | b) & 3 or t.data_ptr() & 7):
        return t, a, b
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.stride(0), t.stride(1)


def _check(who: str, q, k, positions, plan: AxisPlan, norm) -> None:
    if torch.is_grad_enabled() and (grad_needed(q, k) or norm is not None
                                    and grad_needed(norm[0], norm[1])):
        raise RuntimeError(f"{who}: the kernel has no backward; call it under torch.no_grad()")
    qs, ks, D, dev = q.shape, k.shape, plan.head_dim, q.get_device()
    T = qs[0] if qs else 0
    if len(qs) != 3 or len(ks) != 3 or ks[0] != T or qs[2] != D or ks[2] != D:
        raise ValueError(f"{who}: q {tuple(qs)} and k {tuple(ks)} must be [T, heads, {D}]")
    if D % 8 or D > MAX_HEAD_DIM:
        raise ValueError(f"{who}: heads of {D} (multiples of 8 up to {MAX_HEAD_DIM})")
    ps = positions.shape
    if (positions.dtype is not torch.int64 or len(ps) != 2 or ps[1] != T or ps[0] < plan.axes
            or positions.get_device() != dev):
        raise ValueError(f"{who}: positions must be int64 [{plan.axes} axes, {T}] on q's device, "
                         f"got {positions.dtype} {tuple(ps)}")
    if plan.turn.get_device() != dev:
        raise ValueError(f"{who}: the plan is on {plan.turn.device}, q on {q.device}")


def _norm_args(who: str, norm, D: int):
    """Pointers of the norm's weights and its eps."""
    if norm is None:
        return None, None, 0.0
    for w in norm[:2]:
        if w.shape != (D,) or not w.is_contiguous() or w.data_ptr() & 7:
            raise ValueError(f"{who}: norm weights must be contiguous vectors of {D}, 8-byte "
                             "aligned")
    return norm[0].data_ptr(), norm[1].data_ptr(), float(norm[2])


def rotate(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, plan: AxisPlan,
           norm=None) -> tuple[torch.Tensor, torch.Tensor]:
    """q [T, Hq, D] and k [T, Hk, D] turned by positions [axes, T] (int64), as new
    contiguous tensors.  With ``norm = (q_w, k_w, eps)`` each head row is RMS-normed
    first."""
    require_device(q, k, *(norm[:2] if norm is not None else ()))
    _check("rotate", q, k, positions, plan, norm)
    (q, q0, q1), (k, k0, k1) = _ready(q), _ready(k)
    T, Hq, D = q.shape
    Hk = k.shape[1]
    q_out, k_out = (torch.empty(T, h, D, dtype=torch.bfloat16, device=q.device)
                    for h in (Hq, Hk))
    with _lib.device_of(q):
        _lib.call("umic_axial_rope_bf16", q.data_ptr(), k.data_ptr(), q_out.data_ptr(),
                  k_out.data_ptr(), positions.data_ptr(), plan.turn.data_ptr(),
                  plan.axis.data_ptr(), plan.scale, *_norm_args("rotate", norm, D), T, Hq, Hk, D,
                  positions.shape[0], *positions.stride(), q0, q1, k0, k1, Hq * D, D, Hk * D, D,
                  _lib.stream_of(q))
    return q_out, k_out


def rotate_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                  plan: AxisPlan, slots: torch.Tensor, k_pages: torch.Tensor,
                  v_pages: torch.Tensor, norm=None) -> torch.Tensor:
    """``rotate`` of q, with k's rotated rows and v's rows written to ``slots`` (int64
    [T], distinct; one outside the pool writes nothing) of k_pages and v_pages [pages,
    Hk, page_size, D].  Returns the rotated q."""
    require_device(q, k, v, k_pages, v_pages, *(norm[:2] if norm is not None else ()))
    _check("rotate_append", q, k, positions, plan, norm)
    T, Hq, D = q.shape
    Hk = k.shape[1]
    if v.shape != k.shape or torch.is_grad_enabled() and grad_needed(v):
        raise ValueError(f"rotate_append: v {tuple(v.shape)} must be like k {tuple(k.shape)}, "
                         "without a gradient")
    shape, cst = k_pages.shape, k_pages.stride()
    if (len(shape) != 4 or shape != v_pages.shape or shape[1] != Hk or shape[3] != D
            or cst != v_pages.stride() or cst[3] != 1):
        raise ValueError(f"rotate_append: pages {tuple(k_pages.shape)} and {tuple(v_pages.shape)} "
                         f"must be [pages, {Hk}, page_size, {D}] of one layout")
    if (slots.dtype is not torch.int64 or slots.shape != (T,)
            or slots.get_device() != q.get_device() or not slots.is_contiguous()):
        raise ValueError(f"rotate_append: slots must be a contiguous int64 vector of {T} on q's "
                         "device")
    (q, q0, q1), (k, k0, k1), (v, v0, v1) = _ready(q), _ready(k), _ready(v)
    q_out = torch.empty(T, Hq, D, dtype=torch.bfloat16, device=q.device)
    with _lib.device_of(q):
        _lib.call("umic_axial_rope_append_bf16", q.data_ptr(), k.data_ptr(), v.data_ptr(),
                  q_out.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), positions.data_ptr(),
                  plan.turn.data_ptr(), plan.axis.data_ptr(), slots.data_ptr(), plan.scale,
                  *_norm_args("rotate_append", norm, D), T, Hq, Hk, D, positions.shape[0],
                  *positions.stride(), q0, q1, k0, k1, v0, v1, Hq * D, D, cst[0], cst[1], cst[2],
                  shape[0], shape[2], _lib.stream_of(q))
    return q_out
