"""Attention over a cache where scores are far from 0: exact ones (whole numbers that fp32 sums
hold), so that the softmax in 64 bits is known to the last of its differences."""

from __future__ import annotations

import pytest
import torch

import paged_reference as ref
from helpers import bf16_randn
from umic.kernels import attention

pytestmark = pytest.mark.gpu
DEV = "cuda"


def whole(n, S, Hq, Hk, D, seed, far, spread):
    """q, k, v of one request whose scores are far + j, j whole in [-spread, 0]: q = (2^a, 1, 0 ..),
    k = (far 2^-a, j, 0 ..), all of them bf16 values."""
    g = torch.Generator().manual_seed(seed)
    q = torch.zeros(1, Hq, S, D)
    q[..., 0], q[..., 1] = 1024.0, 1.0
    k = torch.zeros(1, Hk, n, D)
    k[..., 0] = far / 1024.0
    j = -torch.randint(0, spread + 1, (1, Hk, n), generator=g).float()
    j[..., torch.randint(0, n, (1,), generator=g)] = 0.0
    k[..., 1] = j
    v = bf16_randn(1, Hk, n, D, gen=g)
    q, k = q.to(torch.bfloat16), k.to(torch.bfloat16)
    assert (k[..., 0].float() == far / 1024.0).all() and (k[..., 1].float() == j).all()
    return q.to(DEV), k.to(DEV), v.to(DEV), j


def softmax(j, v, Hq, S, scale, n):
    """[S, Hq, D] in 64 bits and the kernel's bound: the differences j are exact, their product
    with scale log2(e) is off by 3 2^-24 of itself, which weighs where p > 2^-40, so below 2^-17;
    p by 2^-17 (two bf16 parts, exp2); the sums by (n + 300) 2^-23; numerator and denominator,
    and one rounding to bf16."""
    out, tol = (torch.zeros(S, Hq, v.shape[3], dtype=torch.float64) for _ in range(2))
    Hk = v.shape[1]
    for s in range(S):
        m = n - S + s + 1
        for h in range(Hq):
            g = h // (Hq // Hk)
            x = j[0, g, :m].double() * scale
            p = torch.softmax(x - x.max(), 0)
            vv = v[0, g, :m].double().cpu()
            out[s, h] = p @ vv
            tol[s, h] = 2 * (2.0 ** -16 + (n + 300) * 2.0 ** -23) * (p @ vv.abs())
    return out[None], (tol + 2.0 ** -8 * out.abs() + 1e-37)[None]


SHAPES = [(1, 1, 4, 2, 128), (40, 1, 8, 2, 64), (3100, 1, 8, 2, 128), (5000, 1, 4, 1, 256),
          (300, 3, 8, 2, 128), (700, 40, 4, 2, 128), (2900, 80, 4, 1, 128), (400, 33, 2, 2, 256),
          (400, 20, 2, 2, 64)]


@pytest.mark.parametrize("n,S,Hq,Hk,D", SHAPES)
@pytest.mark.parametrize("far", [2.0 ** 20, -2.0 ** 20, 0.0])
@pytest.mark.parametrize("scale", [0.25, 2.0 ** 13, 2.0 ** 40, 3e30])
def test_far_scores(n, S, Hq, Hk, D, far, scale):
    """Times log2(e), scores of 2^19 to 2^121: above 2^31 the keys of the largest share all."""
    q, k, v, j = whole(n, S, Hq, Hk, D, n + S, far, 30)
    got = attention.cache_attention(q, k, v, n, scale=scale)
    ref.check_attention(got, *softmax(j, v, Hq, S, scale, n))


@pytest.mark.parametrize("n,S,Hq,Hk,D", SHAPES)
@pytest.mark.parametrize("scale", [2.0 ** 127, -2.0 ** 127])
def test_scores_past_fp32_once_scaled(n, S, Hq, Hk, D, scale):
    """The largest scale: every product of a score and it overflows, their differences do not count
    where scores are alike."""
    q, k, v, j = whole(n, S, Hq, Hk, D, n, -2.0 ** 12 if scale > 0 else 2.0 ** 12, 0)
    got = attention.cache_attention(q, k, v, n, scale=scale)
    ref.check_attention(got, *softmax(j, v, Hq, S, 1.0, n))


def test_far_scores_captured():
    """The two-launch forms."""
    for n, S in ((3100, 1), (2900, 40)):
        q, k, v, j = whole(n, S, 8, 2, 128, n, -2.0 ** 20, 30)
        want = attention.cache_attention(q, k, v, n, scale=2.0 ** 13)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = attention.cache_attention(q, k, v, n, scale=2.0 ** 13)
        for _ in range(3):
            out.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
