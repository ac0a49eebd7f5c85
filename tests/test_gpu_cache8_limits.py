"""Calls of the 8-bit cache's operators at their limits: memory that rows share, the largest values,
reads and deals of many workgroups, prompts."""

from __future__ import annotations

import pytest
import torch

import cache8_reference as ref8
import paged_reference as ref
from helpers import bf16_randn
from test_gpu_cache8 import DEV, KINDS, call, filled, new_cache, queries
from umic.kernels import axial, cache8

pytestmark = pytest.mark.gpu


def test_rows_that_share_memory_are_read_not_written():
    cache, table, _, _ = filled("int8", [40], 2, 64, 16, seed=1)
    p = int(table[0, 1])
    thrice = cache8.Pages8(*(t[p:p + 1].expand(3, *t.shape[1:]) for t in cache))
    each, same = (torch.tensor([x], dtype=torch.int32, device=DEV) for x in ([0, 1, 2], [p, p, p]))
    for got, want in zip(cache8.read(thrice, each, 48, 48), cache8.read(cache, same, 48, 48)):
        assert torch.equal(got, want)
    q = queries(1, 1, 4, 64, 1)
    assert torch.equal(call(q, thrice, [48], each), call(q, cache, [48], same))
    x = bf16_randn(4, 2, 64, gen=torch.Generator().manual_seed(1)).to(DEV)
    at = torch.arange(4, device=DEV)
    plan = axial.AxisPlan(torch.ones(32), [0] * 32, device=DEV)
    for bad in (thrice, cache._replace(v=cache.k), cache._replace(v_scale=cache.k_scale)):
        before = [t.clone() for t in cache]
        with pytest.raises(ValueError, match="share memory"):
            cache8.append(x, x, at, bad)
        with pytest.raises(ValueError, match="share memory"):
            cache8.rotate_append(x, x, x, at[None], plan, at, bad)
        for t, was in zip(cache, before):
            assert torch.equal(t.view(torch.uint8), was.view(torch.uint8))


# --- the largest values, and queries past what fp32 holds of their products with codes ---------

MOST = float(torch.finfo(torch.bfloat16).max)


def values_of(cache):
    """(k, v) [pages, Hk, page, D] that the codes stand for: none past bf16's largest number."""
    kc, vc, ks, vs = ref8.numbers(cache)
    return tuple(torch.tensor(ref8.values(c, s)).clamp(-MOST, MOST) for c, s in ((kc, ks), (vc, vs)))


def cache_of(kind, k, v, page=16):
    """A request [n, Hk, D] in pages of its own, and its table."""
    n, Hk, D = k.shape
    pages = -(-n // page)
    cache = new_cache(kind, pages, Hk, page, D)
    cache8.append(k.to(DEV), v.to(DEV), torch.arange(n, device=DEV), cache)
    return cache, torch.arange(pages, dtype=torch.int32, device=DEV)[None]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_the_largest_values_are_finite(kind, D):
    """Numbers that round up to a code past bf16's range are read, and attended to, as the largest."""
    steps = torch.tensor([1.0, 0.99609375, 0.9765625, 0.97265625, 0.5, 0.25])  # of the largest: 255 to 248, 247 ..
    row = torch.cat((steps, -steps, torch.zeros(D - 12))) * MOST
    x = torch.stack((row, row.flip(0), torch.full((D,), MOST)))[:, None].to(torch.bfloat16)  # [3, 1, D]
    x = torch.cat([x[i:i + 1] for i in range(3) for _ in range(16)])  # a block of each
    cache, table = cache_of(kind, x, x)
    k, _ = values_of(cache)
    got = cache8.read(cache, table, 48, 48)
    for y in got:
        assert torch.equal(y[0, 0].double().cpu(), k.flatten(0, 2))
        assert y.isfinite().all()
        err = (y[0, 0].double().cpu() - x[:, 0].double()).abs()
        assert (err <= (2.0 ** -4 * x[:, 0].double().abs() if kind == "e4m3" else 2.0 ** 120)).all()
    for S in (1, 20):  # one key: its own value
        out = call(queries(1, S, 2, D, S) * 0, cache, [1], table)
        assert torch.equal(out[0, -1, 0], got[1][0, 0, 0]) and not out[0, :-1].any()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D,S", [(64, 1), (128, 1), (256, 1), (128, 3), (64, 20), (128, 40), (256, 9)])
def test_large_values_that_rows_do_not_see(kind, D, S):
    """The largest values behind a row leave it as it is; keys of that size that q is 0 for count as
    any other."""
    g = torch.Generator().manual_seed(D + S)
    n, Hk = 150, 2
    k, v = (bf16_randn(n, Hk, D, gen=g) for _ in range(2))
    v[n - 1, 0, ::3] = MOST
    v[n - 1, 1, 1::3] = -MOST
    k[77:79, :, 5] = MOST
    cache, table = cache_of(kind, k, v)
    q = queries(1, S, 4, D, S)
    q[..., 5] = 0
    got = call(q, cache, [n], table)
    want, tol = ref.attention(q, *values_of(cache), [n], table.cpu())
    others = torch.arange(D) % 3 == 2
    for rows in ((got[:, :-1], want[:, :-1], tol[:, :-1]),
                 (got[:, -1:][..., others], want[:, -1:][..., others], tol[:, -1:][..., others])):
        ref.check_attention(*rows)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D,S,Hq", [(64, 1, 4), (128, 1, 8), (256, 1, 2), (128, 20, 4)])
@pytest.mark.parametrize("n", [5, 200, 3000])
def test_large_queries_of_small_keys(kind, D, S, Hq, n):
    """q of 2^122 over keys of 2^-93: scores of ordinary size, but not q times a code."""
    g = torch.Generator().manual_seed(D + n)
    k, v = (bf16_randn(n, 2, D, gen=g) for _ in range(2))
    cache, table = cache_of(kind, (k.float() * 2.0 ** -93).to(torch.bfloat16), v)
    q = (bf16_randn(1, S, Hq, D, gen=g).float() * 2.0 ** 122).to(torch.bfloat16).to(DEV).transpose(1, 2)
    scale = 2.0 ** -29 * D ** -0.5
    got = call(q, cache, [n], table, scale=scale)
    ref.check_attention(got, *ref.attention(q, *values_of(cache), [n], table.cpu(), scale=scale))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_weights_above_one_of_large_values(kind, D):
    """Keys 128 to 159 weigh 2^7 of what came before them, with a value of 2^127 among them: the
    other columns are as they are."""
    g = torch.Generator().manual_seed(D)
    k = torch.zeros(160, 1, D, dtype=torch.bfloat16)
    k[128:, 0, 0] = 5.1875
    v = bf16_randn(160, 1, D, gen=g)
    v[130, 0, 0] = 1.5 * 2.0 ** 127
    cache, table = cache_of(kind, k, v)
    q = torch.zeros(1, 2, 1, D, dtype=torch.bfloat16, device=DEV)
    q[..., 0] = 1.0
    got = call(q, cache, [160], table, scale=1.0)
    want, tol = ref.attention(q, *values_of(cache), [160], table.cpu(), scale=1.0)
    ref.check_attention(got[..., 1:], want[..., 1:], tol[..., 1:])
