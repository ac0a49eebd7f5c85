"""Plain 64-bit forms of the 8-bit cache's operators, for their tests: codes as the whole or
8-bit floating numbers they are, scales as powers of two."""

from __future__ import annotations

import numpy as np
import torch

BLOCK = 16
TYPES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 6, "e4m3": 7}


def code(kind, x):
    """The code nearest to x, ties to even: int8's up to 127; e4m3's of 4 significant bits, in
    steps of 2^-9 at least."""
    if kind == "int8":
        return np.clip(np.rint(x), -127, 127)
    step = np.exp2(np.maximum(np.frexp(x)[1] - 4, -9))
    return np.rint(x / step) * step


def store(kind, codes, scales, x, slots):
    """Rows x [T, H, D] (float64) into codes [P, H, ps, D] and scales [P, H, ps / 16], in place;
    block by block."""
    P, H, ps, _ = codes.shape
    tokens = {}
    for t, s in enumerate(slots):
        if 0 <= s < P * ps:
            tokens.setdefault(s // BLOCK, []).append(t)
    for block, of in tokens.items():
        page, b = divmod(block, ps // BLOCK)
        rows = [slots[t] % BLOCK for t in of]
        first = min(rows)
        for h in range(H):
            new, old = x[of, h], scales[page, h, b]
            part = codes[page, h, b * BLOCK:(b + 1) * BLOCK]
            if not np.isfinite(new).all() or first > 0 and not np.isfinite(old):
                scales[page, h, b] = np.nan
                part[rows] = 0
                continue
            most = np.abs(new).max()
            e = max(int(np.floor(np.log2(most))) - TOP[kind] if most else -100, -100)
            s = max(2.0 ** e, old) if first > 0 else 2.0 ** e
            if first > 0 and s > old:
                part[:first] = code(kind, part[:first] * (old / s))
            part[rows] = code(kind, new / s)
            scales[page, h, b] = s
    return codes, scales


def numbers(cache):
    """(k codes, v codes, k scales, v scales) of a Pages8 as float64 arrays."""
    return tuple(t.float().double().cpu().numpy() for t in cache)


def values(codes, scales):
    """[P, H, ps, D]: code times scale."""
    return codes * np.repeat(scales, BLOCK, axis=2)[..., None]
