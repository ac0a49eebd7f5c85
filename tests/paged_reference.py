"""Plain 64-bit forms of the paged cache's operators, for their tests."""

from __future__ import annotations

import math

import numpy as np
import torch

BF = torch.bfloat16


# --- pages -----------------------------------------------------------------

def plan(kv_len, new, table, ring, cursor, page, tokens, keep=None, delta=None, row=0):
    """(kv_len, cursor, starts, slots, positions, table, ring) after one step, request by
    request; arrays in, new arrays out.  Mirrors the contract of umic_page_plan."""
    R, W, P = len(kv_len), table.shape[1], len(ring)
    table, ring = table.copy(), ring.copy()
    head, free = int(cursor[0]), int(cursor[1])
    slots, positions = np.full(tokens, -1, np.int64), np.zeros(tokens, np.int64)
    starts = np.zeros(R + 1, np.int32)
    kept = [min(max(int(k), 0), int(n)) for k, n in zip(kv_len if keep is None else keep, kv_len)]
    fresh = [max(int(n), 0) for n in new]
    have = [-(-int(n) // page) for n in kv_len]
    need = [-(-(k + n) // page) for k, n in zip(kept, fresh)]
    gave = sum(max(h - n, 0) for h, n in zip(have, need))
    took = sum(max(n - h, 0) for h, n in zip(have, need))
    status = 0
    if (any(n < 0 or n > W * page for n in kv_len) or not 0 <= head < P or not 0 <= free <= P
            or free + gave > P):
        status = 4
    elif any(k + n > W * page for k, n in zip(kept, fresh)):
        status = 2
    elif any(n > row for n in fresh) if row else sum(fresh) > tokens:
        status = 3
    elif took > free + gave:
        status = 1
    if status:
        return (kv_len.copy(), np.array([head, free, 0, status], np.int32), starts, slots, positions,
                table, ring)
    tail = head + free
    for r in range(R):
        for w in range(need[r], have[r]):
            ring[tail % P] = table[r, w]
            tail += 1
    for r in range(R):
        for w in range(have[r], need[r]):
            table[r, w] = ring[head % P]
            head += 1
    for r in range(R):
        at = r * row if row else starts[r]
        for i in range(fresh[r]):
            p = kept[r] + i
            slots[at + i] = int(table[r, p // page]) * page + p % page
            positions[at + i] = p + (0 if delta is None else int(delta[r]))
        starts[r + 1] = starts[r] + fresh[r]
    return (np.array([k + n for k, n in zip(kept, fresh)], np.int32),
            np.array([head % P, tail - head, starts[R], 0], np.int32), starts, slots, positions,
            table, ring)


# --- rotary positions --------------------------------------------------------

def rotate(x, positions, inv_freq, axis, norm_w=None, eps=1e-6, scale=1.0):
    """x [T, H, D] turned, in float64 (cosines of exact angles: positions are integers below
    2^53 / 2^24, inv_freq fp32 values); and |x| |cos| + |partner| |sin|, what errors scale with."""
    x = x.double().cpu()
    if norm_w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * norm_w.double().cpu()
    pos = positions.cpu().double()[torch.as_tensor(axis).cpu().long()].t()  # [T, D/2]
    ang = torch.remainder(pos * inv_freq.double().cpu(), 2 * math.pi)[:, None]
    c, s = ang.cos() * scale, ang.sin() * scale
    a, b = x.chunk(2, dim=-1)
    out = torch.cat((a * c - b * s, b * c + a * s), dim=-1)
    size = torch.cat((a.abs() + b.abs(),) * 2, dim=-1) * abs(scale)
    return out, size


def check_rotated(got, want, size, norm=False):
    """One bf16 rounding (2^-8), and fp32 ahead of it: the sine and cosine to 2^-22, two
    products and a sum (2^-22), with the norm its sum of squares over up to 512 elements, root
    and two products (2^-18 in all at most)."""
    got = got.double().cpu()
    tol = 2.0 ** -8 * want.abs() + size * (2.0 ** -17 if norm else 2.0 ** -20) + 1e-37
    bad = (got - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), (got - want).abs().max())


# --- attention ---------------------------------------------------------------

def dense(cache, table, b, n):
    """Request b's n rows [Hk, n, D]."""
    if table is None:
        return cache[b, :, :n]
    rows = cache.shape[2]
    pages = cache[table[b, :-(-n // rows)].long()]
    return pages.transpose(0, 1).reshape(cache.shape[1], -1, cache.shape[3])[:, :n]


def attention(q, k_cache, v_cache, lens, table=None, q_len=None, causal=True, scale=None, seen=None):
    """[B, S, Hq, D] in float64, and the bound of the kernel's error on each element.

    The kernel's score of a key is an fp32 sum of D exact products: off by at most (D + 4)
    2^-23 of the sum of their sizes X (a unit of the last place for each addition, whichever
    way it rounds, and the scale); its p then by that much and 2^-17 (two bf16 parts, exp2);
    the sums of p and of p v by (n + 300) 2^-23 more each (one addition a key at most, the
    joins).  Numerator and denominator: twice, of sum p |v| / sum p.  Then one rounding to
    bf16, 2^-8 of the value.  seen: [B, n] keys that count (None: all)."""
    B, Hq, S, D = q.shape
    Hk = k_cache.shape[1]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(B, S, Hq, D, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for b in range(B):
        n = int(lens[b])
        fresh = S if q_len is None else max(0, min(S, int(q_len[b])))
        k, v = (dense(c, table, b, n).double().cpu() for c in (k_cache, v_cache))
        for h in range(Hq):
            kh, vh = k[h // (Hq // Hk)], v[h // (Hq // Hk)]
            for s in range(fresh):
                m = min(n, n - fresh + s + 1) if causal else n
                at = torch.arange(max(m, 0))
                if seen is not None:
                    at = at[seen[b][:max(m, 0)]]
                if len(at) == 0:
                    continue
                x = q[b, h, s].double().cpu()
                kk, vv = kh[at], vh[at]
                p = torch.softmax(kk @ x * scale, 0)
                out[b, s, h] = p @ vv
                big = float((kk.abs() @ x.abs()).max()) * abs(scale)
                eps = (D + 4) * 2.0 ** -23 * big + 2.0 ** -17 + (n + 300) * 2.0 ** -23
                tol[b, s, h] = 2 * eps * (p @ vv.abs())
    return out, tol + 2.0 ** -8 * out.abs() + 1e-37


def check_attention(got, want, tol):
    diff = (got.double().cpu() - want).abs()
    bad = ~(diff <= tol)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), float(diff.max()))
