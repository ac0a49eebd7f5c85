"""A paged cache in 8 bits: rows written as codes, read back, and attention over them, against
plain forms in 64 bits (cache8_reference).  Codes, scales and what is read back are compared bit
for bit; attention within the bound that paged_reference.attention derives, as the codes' values
enter its products exactly, in bf16, and scales are powers of two."""

from __future__ import annotations

import math
import random

import numpy as np
import pytest
import torch

import cache8_reference as ref8
import paged_reference as ref
from helpers import bf16_randn
from umic.kernels import attention, axial, cache8, paged

pytestmark = pytest.mark.gpu
DEV = "cuda"
KINDS = ["int8", "e4m3"]


def new_cache(kind, pages, heads, page, D):
    """A pool whose codes and scales are marked: nothing of them may be read."""
    c = cache8.empty(pages, heads, page, D, ref8.TYPES[kind], DEV)
    for t in (c.k, c.v):
        t.view(torch.uint8).fill_(0x7F)  # 127, or NaN
    c.k_scale.fill_(4.0)
    c.v_scale.fill_(4.0)
    return c


def same(got, want):
    assert np.array_equal(got, want, equal_nan=True), np.argwhere(~((got == want) | (got != got)))[:4]


def check_cache(cache, model):
    for got, want in zip(ref8.numbers(cache), model):
        same(got, want)


def append(kind, cache, model, k, v, slots):
    cache8.append(k.to(DEV), v.to(DEV), torch.tensor(slots, device=DEV), cache)
    for i, x in enumerate((k, v)):
        ref8.store(kind, model[i], model[i + 2], x.double().numpy(), slots)
    check_cache(cache, model)


def slots_of(table, page, held, new):
    return [int(table[p // page]) * page + p % page for p in range(held, held + new)]


def spread(g, *shape):
    """Values over many orders of magnitude, row by row and column by column."""
    x = torch.randn(*shape, generator=g)
    rows = torch.exp2(torch.randint(-6, 7, (*shape[:-1], 1), generator=g).float())
    cols = torch.exp2(torch.randint(-3, 4, (shape[-1],), generator=g).float())
    return (x * rows * cols).to(torch.bfloat16)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("Hk,D,page", [(1, 64, 16), (2, 128, 32), (5, 128, 16), (9, 64, 64), (3, 256, 16)])
def test_append(kind, Hk, D, page):
    """Prompts, single tokens and chunks of several requests; each call's codes, scales and the
    rows it leaves alone."""
    g = torch.Generator().manual_seed(D + Hk)
    rng = random.Random(D + page)
    pages, R = 24, 3
    cache = new_cache(kind, pages, Hk, page, D)
    model = list(ref8.numbers(cache))
    ids = torch.randperm(pages, generator=g).view(R, -1)
    held = [0] * R
    for step in range(9):
        new = [rng.choice((0, 1, 1, 2, 15, 16, 17, 40)) for _ in range(R)]
        cap = ids.shape[1] * page
        slots = []
        for r in range(R):
            if held[r] + new[r] > cap or rng.random() < 0.2:
                held[r] = rng.randint(0, held[r])  # drops tokens
            new[r] = min(new[r], cap - held[r])
            slots += slots_of(ids[r], page, held[r], new[r]) + [-1] * rng.randint(0, 2)
            held[r] += new[r]
        k, v = (spread(g, len(slots), Hk, D) for _ in range(2))
        append(kind, cache, model, k, v, slots)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T,lead", [(2049, 3), (2100, 0), (5000, 9)])
def test_append_of_many_tokens(kind, T, lead):
    """More tokens than a workgroup each: runs that begin anywhere in a workgroup's share, and
    single tokens among them."""
    g = torch.Generator().manual_seed(T)
    page, Hk, D = 32, 2, 64
    order = torch.randperm(T // page + 60, generator=g)
    cache = new_cache(kind, len(order), Hk, page, D)
    model = list(ref8.numbers(cache))
    singles = [int(order[i]) * page + 5 for i in range(40)]
    slots = slots_of(order[40:], page, lead, T - 60) + [-1] * 20 + singles
    k, v = (spread(g, T, Hk, D) for _ in range(2))
    append(kind, cache, model, k, v, slots)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [48, 2208])
def test_append_of_interleaved_tokens(kind, T):
    """Two requests' tokens in turn, a third of them without a slot, rows in falling order: those
    of a block stand up to 24 tokens apart."""
    g = torch.Generator().manual_seed(T)
    page, Hk, D = 16, 2, 128
    cache = new_cache(kind, T // page + 4, Hk, page, D)
    model = list(ref8.numbers(cache))
    slots = []
    for i in range(T // 24):  # eight rows of each of two blocks, and eight without a slot
        for j in range(8):
            slots += [(2 * i) * 16 + 9 - j, -1, (2 * i + 1) * 16 + j]
    k, v = (spread(g, T, Hk, D) for _ in range(2))
    append(kind, cache, model, k, v, slots)


@pytest.mark.parametrize("kind", KINDS)
def test_scales_at_their_ends(kind):
    """Zeros, the smallest and largest numbers, powers of two and their neighbours."""
    Hk, D, page = 1, 64, 16
    tiny, huge = 2.0 ** -133, float(torch.finfo(torch.bfloat16).max)
    tops = [0.0, tiny, 2.0 ** -126, 2.0 ** -94, 2.0 ** -93, 2.0 ** -92, 0.9921875, 1.0, 1.0078125,
            1.9921875, 2.0, 448.0, huge, -huge]
    cache = new_cache(kind, len(tops), Hk, page, D)
    model = list(ref8.numbers(cache))
    k = torch.zeros(len(tops), Hk, D)
    steps = torch.linspace(-1, 1, D - 1)
    for i, m in enumerate(tops):
        k[i, 0, 0] = m
        k[i, 0, 1:] = steps * abs(m)
    k = k.to(torch.bfloat16)
    slots = [i * page for i in range(len(tops))]
    append(kind, cache, model, k, -k, slots)
    # and tokens behind them, which raise some scales a long way
    append(kind, cache, model, k.flip(0).contiguous(), k, [s + 1 for s in slots])


@pytest.mark.parametrize("kind", KINDS)
def test_int8_ties_and_the_largest_code(kind):
    """Values half way between codes go to the even one, 127.5 to 127."""
    x = torch.arange(-255, 256).float() / 2
    x = torch.cat((x, torch.zeros(1)))[None, None].view(1, 2, 256).to(torch.bfloat16)
    cache = new_cache(kind, 1, 2, 16, 256)
    model = list(ref8.numbers(cache))
    append(kind, cache, model, x, x, [0])
    if kind == "int8":
        assert int(cache.k.max()) == 127 and int(cache.k.min()) == -127
        assert float(cache.k_scale[0, 0, 0]) == 1.0


@pytest.mark.parametrize("kind", KINDS)
def test_errors_after_growth(kind):
    """Rows written before their block's scale has grown, time after time, are one scale off at
    most (int8); an e4m3 value of normal size is as it was written."""
    D = 128
    cache = new_cache(kind, 1, 1, 16, D)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(16, 1, D, generator=g) * torch.exp2(torch.arange(16) / 2)[:, None, None]
    x = x.to(torch.bfloat16)
    for t in range(16):
        cache8.append(x[t:t + 1].to(DEV), x[t:t + 1].to(DEV), torch.tensor([t], device=DEV), cache)
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    got = cache8.read(cache, table, 16, 16)[0][0, 0].double().cpu()
    want, s = x[:, 0].double(), float(cache.k_scale[0, 0, 0])
    err = (got - want).abs()
    if kind == "int8":
        assert (err[:15] <= s).all() and (err[15] <= s / 2).all()
    else:
        assert (err <= torch.where(want.abs() >= 2.0 ** -6 * s, 2.0 ** -4 * want.abs(), 2.0 ** -9 * s)).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_values_that_are_not_finite(kind, bad):
    """Their block of their head is NaN, until it is begun anew; its neighbours are as ever."""
    g = torch.Generator().manual_seed(2)
    cache = new_cache(kind, 4, 3, 32, 128)
    model = list(ref8.numbers(cache))
    k, v = (bf16_randn(40, 3, 128, gen=g) for _ in range(2))
    k[17, 1, 5] = bad
    v[33, 2, 127] = bad
    append(kind, cache, model, k, v, list(range(40)))
    append(kind, cache, model, k[:9], v[:9], list(range(40, 49)))   # the open block stays NaN
    table = torch.tensor([[0, 1]], dtype=torch.int32, device=DEV)
    for got, x, hit in zip(cache8.read(cache, table, 49, 64), model[:2], ((1, 16), (2, 32))):
        want = torch.zeros(3, 64, dtype=torch.bool)
        want[hit[0], hit[1]:hit[1] + 16] = True
        assert torch.equal(torch.isnan(got[0]).any(-1).cpu(), want & (torch.arange(64) < 49))
    append(kind, cache, model, k[:5], v[:5], list(range(32, 37)))   # begun anew


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [1, 5, 77, 2200])
@pytest.mark.parametrize("Hq,Hk,D", [(32, 8, 128), (14, 2, 64), (4, 3, 256)])
@pytest.mark.parametrize("norm", [False, True])
def test_rotate_append(kind, T, Hq, Hk, D, norm):
    """q against the formula in 64 bits; the cache, to the bit, that of the same rows rotated as q
    and appended."""
    g = torch.Generator().manual_seed(T + D)
    q, k, v = (bf16_randn(T, h, D, gen=g).to(DEV) for h in (Hq, Hk, Hk))
    inv, axis = (1e4 ** (-torch.arange(D // 2) / (D // 2))).float(), torch.arange(D // 2) % 3
    plan = axial.AxisPlan(inv, axis, 1.25, DEV)
    pos = torch.randint(-9, 40000, (3, T), generator=g).to(DEV)
    qw, kw = (bf16_randn(D, scale=0.1, shift=1.0, gen=g).to(DEV) for _ in range(2))
    one, two, spare = (new_cache(kind, T // 16 + 3, Hk, 16, D) for _ in range(3))
    slots = torch.arange(T, device=DEV) + 21
    got = cache8.rotate_append(q, k, v, pos, plan, slots, one, (qw, kw, 1e-5) if norm else None)
    ref.check_rotated(got, *ref.rotate(q, pos, inv, axis, qw if norm else None, 1e-5, 1.25), norm)
    turned = cache8.rotate_append(k, k, v, pos, plan, slots, spare, (kw, kw, 1e-5) if norm else None)
    cache8.append(turned, v, slots, two)
    for a, b in zip(one, two):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("kind", KINDS)
def test_append_of_views(kind):
    """Rows of a packed projection, rows that are not of 16-byte chunks, token-major positions,
    pages with gaps between them; slots outside the pool write nothing."""
    g = torch.Generator().manual_seed(4)
    T, Hk, D = 21, 2, 64
    qkv = bf16_randn(T, 8, D, gen=g).to(DEV)
    odd = bf16_randn(T, Hk, D + 1, gen=g).to(DEV)[..., 1:]
    room = torch.zeros(5, 2, 3, 32, D + 16, dtype=torch.uint8, device=DEV)
    dt = ref8.TYPES[kind]
    scales = torch.zeros(5, 2, 3, 2, device=DEV)
    cache = cache8.Pages8(room[:, 0, :2, :, :D].view(dt), room[:, 1, :2, :, :D].view(dt),
                          scales[:, 0, :2], scales[:, 1, :2])
    slots = list(range(30, 30 + T))
    slots[2], slots[9], slots[20] = -1, 5 * 32, 1 << 40
    model = list(ref8.numbers(cache))
    cache8.append(qkv[:, 6:], odd, torch.tensor(slots, device=DEV), cache)
    for i, x in enumerate((qkv[:, 6:], odd)):
        ref8.store(kind, model[i], model[i + 2], x.double().cpu().numpy(), slots)
    check_cache(cache, model)
    assert not room[:, :, 2].any() and not room[..., D:].any() and not scales[:, :, 2].any()


# --- reading ------------------------------------------------------------------

def filled(kind, lens, Hk, D, page, seed=0, slack=3):
    """A cache of requests of these lengths, its table (-1 past their pages), and its values
    [pages, Hk, page, D]; whatever lies past a length is marked, and scales of blocks without a
    token are NaN."""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // page) for n in lens]
    ids = torch.randperm(sum(counts) + slack, generator=g)
    cache = new_cache(kind, len(ids), Hk, page, D)
    cache.k_scale.fill_(math.nan)
    cache.v_scale.fill_(math.nan)
    table = torch.full((len(lens), max(counts) + 1), -1, dtype=torch.int32)
    at, slots = 0, []
    for b, c in enumerate(counts):
        table[b, :c] = ids[at:at + c]
        at += c
        slots += slots_of(table[b], page, 0, lens[b])
    k, v = (bf16_randn(len(slots), Hk, D, gen=g) for _ in range(2))
    k *= torch.exp2(torch.randint(-2, 3, (D,), generator=g).float()).to(torch.bfloat16)
    if slots:
        cache8.append(k.to(DEV), v.to(DEV), torch.tensor(slots, device=DEV), cache)
    kc, vc, ks, vs = ref8.numbers(cache)
    return cache, table.to(DEV), torch.tensor(ref8.values(kc, ks)), torch.tensor(ref8.values(vc, vs))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("Hk,D,page", [(2, 64, 16), (8, 128, 64), (1, 256, 32)])
def test_read(kind, Hk, D, page):
    lens = [1, 0, 16, 33, 200]
    cache, table, k, v = filled(kind, lens, Hk, D, page, seed=D)
    starts = [0, 5, 3, 40, 190]
    n, start = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (lens, starts))
    for rows, begin in ((200, None), (7, None), (37, start), (0, start)):
        got = cache8.read(cache, table, n, rows, start=begin)
        for x, want in zip(got, (k, v)):
            assert x.shape == (5, Hk, rows, D) and x.dtype is torch.bfloat16
            for b, m in enumerate(lens):
                at = 0 if begin is None else starts[b]
                dense = torch.zeros(Hk, rows, D, dtype=torch.float64)
                part = ref.dense(want, table.cpu(), b, m)[:, at:at + rows]
                dense[:, :part.shape[1]] = part
                assert torch.equal(x[b].double().cpu(), dense), (rows, b)
    one = cache8.read(cache, table[4:], 200, 200)
    assert torch.equal(one[0][0], cache8.read(cache, table, n, 200)[0][4])


def test_read_of_what_is_not_there():
    """Lengths past the table, negative ones and starts, pages outside the pool."""
    cache, table, k, _ = filled("int8", [48, 48], 2, 64, 16, seed=2)
    table = table[:, :3].contiguous()
    table[0, 1], table[1, 0], table[1, 2] = -1, cache.k.shape[0], -(1 << 31)
    n = torch.tensor([1 << 30, 48], dtype=torch.int32, device=DEV)
    start = torch.tensor([-7, 3], dtype=torch.int32, device=DEV)
    got = cache8.read(cache, table, n, 60, start=start)[0].double().cpu()
    want = torch.zeros(2, 2, 60, 64, dtype=torch.float64)
    want[0, :, :16], want[0, :, 32:48] = k[int(table[0, 0])], k[int(table[0, 2])]
    want[1, :, 13:29] = k[int(table[1, 1])]
    assert torch.equal(got, want)
    n = torch.tensor([-1, 0], dtype=torch.int32, device=DEV)
    assert not any(x.any() for x in cache8.read(cache, table, n, 20))
    assert not any(x.any() for x in cache8.read(cache, table, 0, 20))


# --- attention ----------------------------------------------------------------

def queries(B, S, Hq, D, seed):
    g = torch.Generator().manual_seed(seed + 1000)
    return bf16_randn(B, S, Hq, D, scale=1.5, gen=g).to(DEV).transpose(1, 2)


def call(q, cache, lens, table, **kw):
    return cache8.attention(q, cache, torch.tensor(lens, dtype=torch.int32, device=DEV), table, **kw)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("Hq,Hk,D", [(8, 2, 128), (4, 4, 64), (4, 1, 256), (14, 2, 64), (32, 2, 128)])
def test_single_tokens(kind, page, Hq, Hk, D):
    lens = [1, 0, 15, 16, 17, 31, 33, 127, 128, 129, 300, 1025]
    cache, table, k, v = filled(kind, lens, Hk, D, page, seed=D + page)
    q = queries(len(lens), 1, Hq, D, page)
    got = call(q, cache, lens, table)
    ref.check_attention(got, *ref.attention(q, k, v, lens, table.cpu()))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [1, 2, 40, 128, 3100])
def test_one_length_for_all(kind, n):
    cache, table, k, v = filled(kind, [n] * 2, 2, 128, 32, seed=n)
    q = queries(2, 1, 8, 128, n)
    got = cache8.attention(q, cache, n, table)
    ref.check_attention(got, *ref.attention(q, k, v, [n] * 2, table.cpu()))
    assert torch.equal(got, call(q, cache, [n] * 2, table))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("S,Hq,Hk,D", [(2, 8, 2, 128), (5, 4, 4, 64), (7, 8, 2, 128), (32, 4, 1, 128),
                                       (9, 6, 1, 256), (70, 2, 2, 64), (33, 4, 2, 128)])
@pytest.mark.parametrize("causal", [True, False])
def test_several_tokens(kind, S, Hq, Hk, D, causal):
    lens = [S, S + 1, 3 * S + 130, 1, 0]  # the last two shorter than their new tokens
    cache, table, k, v = filled(kind, lens, Hk, D, 16, seed=S)
    q = queries(5, S, Hq, D, S)
    got = call(q, cache, lens, table, causal=causal)
    ref.check_attention(got, *ref.attention(q, k, v, lens, table.cpu(), causal=causal))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("S,Hq,Hk,D,page", [(80, 8, 2, 128, 64), (70, 14, 2, 64, 16), (40, 4, 2, 256, 128)])
def test_several_row_blocks(kind, S, Hq, Hk, D, page):
    """More query rows than a workgroup has, over requests that many workgroups share; some
    with fewer new tokens than rows."""
    lens, fresh = [2900, S, 0, S + 31, 3 * S, 1500], [S, S, 0, S // 3, 0, 5]
    cache, table, k, v = filled(kind, lens, Hk, D, page, seed=S)
    q = queries(len(lens), S, Hq, D, S)
    n = torch.tensor(fresh, dtype=torch.int32, device=DEV)
    got = call(q, cache, lens, table, q_len=n)
    ref.check_attention(got, *ref.attention(q, k, v, lens, table.cpu(), q_len=fresh))
    for b, m in enumerate(fresh):
        assert not got[b, m:].any()
    got = call(q, cache, lens, table, causal=False)
    ref.check_attention(got, *ref.attention(q, k, v, lens, table.cpu(), causal=False))


def test_many_requests_of_all_lengths():
    rng = random.Random(4)
    lens = [rng.choice((0, 1, 130, rng.randint(0, 700))) for _ in range(610)]
    cache, table, k, v = filled("e4m3", lens, 1, 64, 16, seed=4)
    q = queries(610, 1, 2, 64, 4)
    ref.check_attention(call(q, cache, lens, table), *ref.attention(q, k, v, lens, table.cpu()))


@pytest.mark.parametrize("S", [1, 9])
def test_lengths_and_pages_that_are_not_there(S):
    lens = [200, 90]
    cache, table, k, v = filled("int8", lens, 2, 128, 16, seed=3)
    q = queries(2, S, 8, 128, 3)
    seen = torch.ones(2, 200, dtype=torch.bool)
    good = table.cpu()
    for b, w, bad in ((0, 0, -1), (0, 5, cache.k.shape[0]), (0, 12, 1 << 30), (1, 3, -(1 << 31))):
        table[b, w] = bad
        seen[b, 16 * w:16 * w + 16] = False
    got = call(q, cache, lens, table)
    ref.check_attention(got, *ref.attention(q, k, v, lens, good, seen=seen))
    out = torch.full((2, S, 8, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    assert not call(q, cache, [0, -5], table, out=out).any()
    cut = good[:, :3].contiguous().to(DEV)
    assert torch.equal(call(q, cache, [1 << 30, 48], cut), call(q, cache, [48, 48], cut))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("D,S", [(128, 1), (128, 3), (64, 40), (256, 9)])
def test_blocks_that_read_as_nan(kind, which, D, S):
    """Rows that see one of the block's keys are NaN, for its head; the others as without it."""
    lens, Hq, Hk = [150, 150], 4, 2
    cache, table, k, v = filled(kind, lens, Hk, D, 16, seed=S)
    q = queries(2, S, Hq, D, S)
    want, tol = ref.attention(q, k, v, lens, table.cpu())
    block = 9  # of the last tokens: keys 144 to 149
    scale = cache.k_scale if which == "k" else cache.v_scale
    scale[int(table[0, block]), 1, 0] = math.nan
    got = call(q, cache, lens, table).cpu()
    hit = torch.zeros(2, S, Hq, dtype=torch.bool)
    for s in range(S):
        hit[0, s, 2:] = 150 - S + s >= 16 * block
    assert torch.isnan(got[hit]).all()
    hit = hit[..., None].expand(got.shape)
    ref.check_attention(torch.where(hit, 0, got), torch.where(hit, 0, want), tol)


@pytest.mark.parametrize("S", [1, 20])
def test_large_scores_and_scale(S):
    lens = [777]
    cache, table, k, v = filled("int8", lens, 2, 128, 64, seed=7)
    q = queries(1, S, 4, 128, 7) * 40
    for scale in (1.0, -0.5, 0.0):
        got = call(q, cache, lens, table, scale=scale)
        ref.check_attention(got, *ref.attention(q, k, v, lens, table.cpu(), scale=scale))


def test_views_of_queries_and_outputs():
    g = torch.Generator().manual_seed(1)
    cache, table, k, v = filled("e4m3", [70, 20], 2, 64, 16, seed=3)
    qkv = bf16_randn(2, 3, 12, 64, gen=g).to(DEV)
    q = qkv[:, :, 1:9].transpose(1, 2)
    room = torch.full((2, 3, 9, 72), 5.0, dtype=torch.bfloat16, device=DEV)
    out = room[:, :, :8, :64]
    assert call(q, cache, [70, 20], table, out=out) is out
    ref.check_attention(out, *ref.attention(q, k, v, [70, 20], table.cpu()))
    assert (room[:, :, 8] == 5).all() and (room[..., 64:] == 5).all()
    wide = torch.full((2, 40), -1, dtype=torch.int32, device=DEV)
    wide[:, 7:7 + table.shape[1]] = table
    odd = bf16_randn(2, 8, 1, 65, gen=g).to(DEV)[..., 1:]
    got = call(odd, cache, [70, 20], wide[:, 7:7 + table.shape[1]])
    ref.check_attention(got, *ref.attention(odd, k, v, [70, 20], table.cpu()))


def test_offsets_past_32_bits():
    """Pages more than 2^31 codes into the pool."""
    page, Hk, D = 64, 8, 128
    pages = (1 << 31) // (page * Hk * D) + 3
    cache = cache8.Pages8(*(torch.zeros(pages, Hk, page, D, dtype=torch.int8, device=DEV) for _ in range(2)),
                          *(torch.ones(pages, Hk, page // 16, device=DEV) for _ in range(2)))
    ids = [0, pages - 1, pages // 2, pages - 2]
    table = torch.tensor([ids], dtype=torch.int32, device=DEV)
    g = torch.Generator().manual_seed(2)
    k, v = (bf16_randn(250, Hk, D, gen=g).to(DEV) for _ in range(2))
    slots = torch.tensor(slots_of(ids, page, 0, 250), device=DEV)
    cache8.append(k, v, slots, cache)
    rows = cache8.read(cache, table, 250, 250)
    for x, y in zip(rows, (k, v)):
        assert ((x[0].transpose(0, 1).float() - y.float()).abs() <= y.float().abs().max() / 64).all()
    q = bf16_randn(1, 8, 1, D, gen=g).to(DEV)
    got = cache8.attention(q, cache, 250, table)
    ref.check_attention(got, *ref.attention(q, *(x.double() for x in rows), [250]))


# --- streams, graphs, a run of all ---------------------------------------------

def test_results_repeat_and_streams_agree():
    lens = [900, 33, 0, 2500]
    cache, table, _, _ = filled("int8", lens, 2, 128, 16, seed=5)
    q = queries(4, 1, 8, 128, 5)
    want = call(q, cache, lens, table)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    torch.cuda.synchronize()
    for i in range(6):  # two calls at once
        with torch.cuda.stream(side[i % 2]):
            got.append(cache8.attention(q, cache, n, table))
    torch.cuda.synchronize()
    for o in got:
        assert torch.equal(o, want)


@pytest.mark.parametrize("S", [1, 20])
def test_captured_steps(S):
    """Two captured steps (rows written, read and attended to), replayed at once, against eager
    calls on copies."""
    lens = [[300, 41], [64, 1111]]
    Hq, Hk, D, page = 8, 2, 128, 16
    g = torch.Generator().manual_seed(S)
    plan = axial.AxisPlan(torch.ones(D // 2), [0] * (D // 2), device=DEV)
    steps, graphs, outs = [], [], []
    for i, x in enumerate(lens):
        cache, table, _, _ = filled(KINDS[i], [m + 3 * S for m in x], Hk, D, page, seed=i)
        q, k, v = (bf16_randn(2 * S, h, D, gen=g).to(DEV) for h in (Hq, Hk, Hk))
        pos = torch.zeros(1, 2 * S, dtype=torch.int64, device=DEV)
        slots = torch.zeros(2 * S, dtype=torch.int64, device=DEV)
        n = torch.tensor(x, dtype=torch.int32, device=DEV)
        steps.append((cache, table, q, k, v, pos, slots, n))

    def step(cache, table, q, k, v, pos, slots, n):
        q = cache8.rotate_append(q, k, v, pos, plan, slots, cache)
        return (cache8.attention(q.view(2, S, Hq, D).transpose(1, 2), cache, n, table),
                *cache8.read(cache, table, n, 40))

    def at(i, move):
        table, n = steps[i][1].tolist(), [m + move * S for m in lens[i]]
        return [s for b in range(2) for s in slots_of(table[b], page, n[b] - S, S)], n

    for i, s in enumerate(steps):
        s[6].copy_(torch.tensor(at(i, 1)[0]))
        graph = torch.cuda.CUDAGraph()
        step(*s)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            outs.append(step(*s))
        graphs.append(graph)
    side = [torch.cuda.Stream() for _ in graphs]
    for move in (1, 2, 3):
        copies = []
        for i, s in enumerate(steps):
            where, n = at(i, move)
            s[6].copy_(torch.tensor(where))
            s[7].copy_(torch.tensor(n, dtype=torch.int32))
            s[3].mul_(1.5)
            copies.append((cache8.Pages8(*(t.clone() for t in s[0])), *s[1:]))
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, side):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for s, copy, out in zip(steps, copies, outs):
            for a, b in zip(out, step(*copy)):
                assert torch.equal(a, b)
            for a, b in zip(s[0], copy[0]):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("kind", KINDS)
def test_served_together(kind):
    """A server's steps, as a user runs them: pages planned, keys rotated into them, attended to;
    requests end and begin.  Against a model of the pool in 64 bits."""
    rng = random.Random(8)
    R, W, page, Hq, Hk, D, P = 5, 20, 16, 8, 2, 128, 90
    i32 = dict(dtype=torch.int32, device=DEV)
    n, table = torch.zeros(R, **i32), torch.zeros(R, W, **i32)
    ring, cursor = torch.arange(P, **i32), torch.tensor([0, P, 0, 0], **i32)
    cache = new_cache(kind, P, Hk, page, D)
    model = list(ref8.numbers(cache))
    inv = (1e4 ** (-torch.arange(D // 2) / (D // 2))).float()
    plan = axial.AxisPlan(inv, torch.arange(D // 2) % 3, device=DEV)
    g = torch.Generator().manual_seed(3)
    for step in range(8):
        keep = [0 if rng.random() < 0.3 else 1 << 30 for _ in range(R)]
        S = rng.choice((1, 1, 30))
        new = [rng.randint(0, S) if S > 1 else 1 for _ in range(R)]
        t = paged.plan_pages(n, torch.tensor(new, **i32), table, ring, cursor, page, R * S,
                             keep=torch.tensor(keep, **i32), row=S)
        assert t.cursor.tolist()[3] == paged.PLAN_OK
        n, cursor = t.kv_len, t.cursor
        q, k, v = (bf16_randn(R * S, h, D, gen=g).to(DEV) for h in (Hq, Hk, Hk))
        pos = t.positions.expand(3, -1)
        q = cache8.rotate_append(q, k, v, pos, plan, t.slots, cache)
        got = cache8.attention(q.view(R, S, Hq, D).transpose(1, 2), cache, n, table,
                               q_len=torch.tensor(new, **i32))
        spare = cache8.empty(R * S // 16 + 1, Hk, 16, D, ref8.TYPES[kind], DEV)
        turned = cache8.rotate_append(k, k, v, pos, plan, torch.arange(R * S, device=DEV), spare)
        for i, x in enumerate((turned, v)):
            ref8.store(kind, model[i], model[i + 2], x.double().cpu().numpy(), t.slots.tolist())
        check_cache(cache, model)
        dense = [torch.tensor(ref8.values(model[i], model[i + 2])) for i in (0, 1)]
        ref.check_attention(got, *ref.attention(q.view(R, S, Hq, D).transpose(1, 2), *dense, n.tolist(),
                                                table.cpu(), q_len=new))
