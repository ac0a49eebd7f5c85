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


# --- launches of many workgroups -----------------------------------------------

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_reads_on_both_sides_of_two_rows_a_thread(kind, D):
    """Up to where a read's workgroups come to eight a CU, its threads have one row each, then two:
    the last one row, the next one, and odd ones; requests that end inside, starts, pages that are
    not there."""
    B, Hk, page = 4, 64, 16
    per = 2 * (256 // (D // 8))  # rows of a workgroup whose threads have two
    groups = -(-8 * torch.cuda.get_device_properties(0).multi_processor_count // (2 * B * Hk))
    edge = (groups - 1) * per
    lens = [edge + 40, edge - 3, 5, 0]
    cache, table, k, v = filled(kind, lens, Hk, D, page, seed=D)
    table[0, 1], table[1, 2] = -1, cache.k.shape[0]
    at = table.cpu()
    starts = [11, 0, 3, 9]
    n, start = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (lens, starts))
    for rows in (edge, edge + 1, edge + per // 2 + 1, edge + per - 1, edge + per, edge + per + 3):
        for begin in (None, start):
            got = cache8.read(cache, table, n, rows, start=begin)
            for x, pool in zip(got, (k, v)):
                for b, m in enumerate(lens):
                    first = 0 if begin is None else starts[b]
                    want = torch.zeros(Hk, rows, D, dtype=torch.float64)
                    for i in range(first // page, -(-m // page)):
                        p, lo, hi = int(at[b, i]), i * page - first, min((i + 1) * page, m) - first
                        if 0 <= p < len(pool) and lo < rows:
                            part = pool[p][:, max(-lo, 0):hi - lo][:, :rows - max(lo, 0)]
                            want[:, max(lo, 0):max(lo, 0) + part.shape[1]] = part
                    assert torch.equal(x[b].double().cpu(), want), (rows, b, first)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("Hq,Hk,D,lens", [(4, 2, 64, [120001, 0, 50003, 1]), (3, 1, 256, [90001, 80003]),
                                          (16, 1, 64, [250000])])
def test_single_tokens_over_many_keys(kind, Hq, Hk, D, lens):
    """A segment in some hundred parts, of a launch that fills the chip."""
    cache, table, k, v = filled(kind, lens, Hk, D, 64, seed=D)
    q = queries(len(lens), 1, Hq, D, D)
    got = call(q, cache, lens, table)
    ref.check_attention(got, *ref.attention(q, k, v, lens, table.cpu()))
    assert torch.equal(got, call(q, cache, lens, table))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("S,Hq,Hk,D", [(300, 8, 2, 128), (1030, 2, 1, 64), (200, 2, 1, 256)])
def test_prompts(kind, S, Hq, Hk, D):
    """A prompt over itself, and one behind what its request holds."""
    lens = [S, 2 * S + 77]
    cache, table, k, v = filled(kind, lens, Hk, D, 32, seed=S)
    q = queries(2, S, Hq, D, S)
    ref.check_attention(call(q, cache, lens, table), *ref.attention(q, k, v, lens, table.cpu()))


@pytest.mark.parametrize("kind", KINDS)
def test_a_long_prompt(kind):
    """3100 tokens over themselves: some of its rows, by themselves."""
    n, Hq, Hk, D = 3100, 8, 2, 128
    cache, table, k, v = filled(kind, [n], Hk, D, 64, seed=n)
    q = queries(1, n, Hq, D, n)
    got = call(q, cache, [n], table)
    for s in (0, 1, 15, 16, 31, 32, 127, 128, 1000, 1549, 2047, 2048, 3070, 3092, 3098, 3099):
        ref.check_attention(got[:, s:s + 1], *ref.attention(q[:, :, s:s + 1], k, v, [s + 1], table.cpu()))


# --- rotated keys ----------------------------------------------------------------

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [5, 300, 2200])
@pytest.mark.parametrize("Hk,D", [(2, 128), (3, 64), (1, 256)])
@pytest.mark.parametrize("norm", [False, True])
def test_rotated_keys_against_the_formula(kind, T, Hk, D, norm):
    """k's rows as they are read back, against the rotation in 64 bits: off by check_rotated's
    bound, their rounding to bf16 in it, and then by half a step of the codes: half a scale
    (int8; a whole one for what rounds to 128 codes and more, held as 127), 2^-4 of the value or
    2^-10 scales (e4m3).  The scale is that of the block's largest value, one up or down where
    rounding crosses a power of two."""
    g = torch.Generator().manual_seed(T + D)
    q, k, v = (bf16_randn(T, Hk, D, gen=g).to(DEV) for _ in range(3))
    inv, axis = (1e4 ** (-torch.arange(D // 2) / (D // 2))).float(), torch.arange(D // 2) % 3
    plan = axial.AxisPlan(inv, axis, 1.25, DEV)
    pos = torch.randint(-9, 40000, (3, T), generator=g).to(DEV)
    qw, kw = (bf16_randn(D, scale=0.1, shift=1.0, gen=g).to(DEV) for _ in range(2))
    cache = new_cache(kind, T // 16 + 1, Hk, 16, D)
    at = torch.randperm(T, generator=g)
    cache8.rotate_append(q, k, v, pos, plan, at.to(DEV), cache, (qw, kw, 1e-5) if norm else None)
    table = torch.arange(cache.k.shape[0], dtype=torch.int32, device=DEV)[None]
    got = cache8.read(cache, table, T, T)[0][0].transpose(0, 1).double().cpu()[at]  # [T, Hk, D]
    want, size = ref.rotate(k, pos, inv, axis, kw if norm else None, 1e-5, 1.25)
    tol = 2.0 ** -8 * want.abs() + size * (2.0 ** -17 if norm else 2.0 ** -20) + 1e-37
    scale = cache.k_scale[..., 0].double().cpu()[at // 16][..., None]  # [T, Hk, 1]
    step = scale / 2 if kind == "int8" else torch.maximum(2.0 ** -4 * (want.abs() + tol), 2.0 ** -10 * scale)
    if kind == "int8":
        step = torch.where(want.abs() + tol > 127.5 * scale, scale, step)
    bad = (got - want).abs() > tol + step
    assert not bad.any(), (int(bad.sum()), float((got - want).abs().max()))
    lo, hi = torch.zeros(2, cache.k.shape[0], Hk, dtype=torch.float64)
    for t in range(T):
        b = int(at[t]) // 16
        lo[b] = torch.maximum(lo[b], (want[t].abs() - tol[t]).amax(-1))
        hi[b] = torch.maximum(hi[b], (want[t].abs() + tol[t]).amax(-1))
    used = hi[:, 0] > 0
    e = torch.log2(cache.k_scale[..., 0].double().cpu())[used] + ref8.TOP[kind]
    assert (e >= torch.floor(torch.log2(lo[used]))).all() and (e <= torch.floor(torch.log2(hi[used]))).all()
