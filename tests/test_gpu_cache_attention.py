"""Attention over a paged or contiguous cache (umic_cache_attention_bf16) against softmax in
64 bits, within the bound that paged_reference.attention derives."""

from __future__ import annotations

import math
import random

import pytest
import torch

import paged_reference as ref
from helpers import bf16_randn
from umic.cache import KVArena
from umic.kernels import attention, axial, paged

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(lens, S, Hq, Hk, D, page, seed=0, slack=3):
    """q [B, Hq, S, D] (a transposed view) and the cache of requests of these lengths; whatever
    lies past a length is NaN."""
    g = torch.Generator().manual_seed(seed)
    B = len(lens)
    q = bf16_randn(B, S, Hq, D, scale=1.5, gen=g).to(DEV).transpose(1, 2)
    if not page:
        shape, table = (B, Hk, max(lens) + slack, D), None
    else:
        counts = [-(-n // page) for n in lens]
        ids = torch.randperm(sum(counts) + slack, generator=g)
        table = torch.full((B, max(counts) + 1), -1, dtype=torch.int32)
        at = 0
        for b, c in enumerate(counts):
            table[b, :c] = ids[at:at + c]
            at += c
        shape, table = (len(ids), Hk, page, D), table.to(DEV)
    k, v = (bf16_randn(*shape, gen=g) for _ in range(2))
    live = torch.zeros(shape[0], shape[2], dtype=torch.bool)
    for b, n in enumerate(lens):
        if page:
            for j in range(n):
                live[int(table[b, j // page]), j % page] = True
        else:
            live[b, :n] = True
    dead = ~live[:, None, :, None].expand(shape)
    k[dead], v[dead] = float("nan"), float("nan")
    return q, k.to(DEV), v.to(DEV), table


def call(q, k, v, lens, table, **kw):
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    return attention.cache_attention(q, k, v, n, table=table, **kw)


@pytest.mark.parametrize("page", [0, 16, 64])
@pytest.mark.parametrize("Hq,Hk,D", [(8, 2, 128), (4, 4, 64), (4, 1, 256), (14, 2, 64), (32, 1, 128)])
def test_single_tokens(page, Hq, Hk, D):
    lens = [1, 0, 15, 16, 17, 31, 33, 127, 128, 129, 300, 1025]
    q, k, v, table = make(lens, 1, Hq, Hk, D, page, seed=D + page)
    got = call(q, k, v, lens, table)
    ref.check_attention(got, *ref.attention(q, k, v, lens, table))


@pytest.mark.parametrize("n", [1, 2, 40, 128, 3100])
@pytest.mark.parametrize("page", [0, 32])
def test_one_length_for_all(n, page):
    q, k, v, table = make([n] * 2, 1, 8, 2, 128, page, seed=n)
    got = attention.cache_attention(q, k, v, n, table=table)
    ref.check_attention(got, *ref.attention(q, k, v, [n] * 2, table))
    assert torch.equal(got, call(q, k, v, [n] * 2, table))


@pytest.mark.parametrize("S,Hq,Hk,D", [(2, 8, 2, 128), (5, 4, 4, 64), (7, 8, 2, 128), (32, 4, 1, 128),
                                       (9, 6, 1, 256), (70, 2, 2, 64), (33, 4, 2, 128)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("page", [0, 16])
def test_several_tokens(S, Hq, Hk, D, causal, page):
    lens = [S, S + 1, 3 * S + 130, 1, 0]  # the last two shorter than their new tokens
    q, k, v, table = make(lens, S, Hq, Hk, D, page, seed=S)
    got = call(q, k, v, lens, table, causal=causal)
    ref.check_attention(got, *ref.attention(q, k, v, lens, table, causal=causal))


@pytest.mark.parametrize("causal", [True, False])
def test_fewer_new_tokens_than_rows(causal):
    S, lens, fresh = 6, [200, 9, 64, 70, 5], [6, 0, 1, 3, 5]
    q, k, v, table = make(lens, S, 8, 4, 128, 32, seed=9)
    n = torch.tensor(fresh, dtype=torch.int32, device=DEV)
    got = call(q, k, v, lens, table, q_len=n, causal=causal)
    want, tol = ref.attention(q, k, v, lens, table, q_len=fresh, causal=causal)
    ref.check_attention(got, want, tol)
    for b, m in enumerate(fresh):
        assert not got[b, m:].any()


@pytest.mark.parametrize("S,Hq,Hk,D,page", [(80, 8, 2, 128, 64), (70, 14, 2, 64, 16), (40, 4, 2, 256, 128),
                                            (257, 2, 2, 128, 0)])
def test_several_row_blocks(S, Hq, Hk, D, page):
    """More query rows than a workgroup has, over requests that many workgroups share."""
    lens, fresh = [2900, S, 0, S + 31, 3 * S, 1500], [S, S, 0, S // 3, 0, 5]
    q, k, v, table = make(lens, S, Hq, Hk, D, page, seed=S)
    n = torch.tensor(fresh, dtype=torch.int32, device=DEV)
    got = call(q, k, v, lens, table, q_len=n)
    ref.check_attention(got, *ref.attention(q, k, v, lens, table, q_len=fresh))
    got = call(q, k, v, lens, table, causal=False)
    ref.check_attention(got, *ref.attention(q, k, v, lens, table, causal=False))


def test_many_requests_of_all_lengths():
    rng = random.Random(4)
    lens = [rng.choice((0, 1, 130, rng.randint(0, 700))) for _ in range(610)]
    q, k, v, table = make(lens, 1, 2, 1, 64, 16, seed=4)
    ref.check_attention(call(q, k, v, lens, table), *ref.attention(q, k, v, lens, table))


def test_empty_cache_gives_zeros():
    q, k, v, table = make([5, 5], 2, 4, 2, 128, 16)
    out = torch.full((2, 2, 4, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    assert not call(q, k, v, [0, 0], table, out=out).any()
    assert not attention.cache_attention(q, k, v, 0, table=table).any()
    none = k[:, :, :0]
    assert not attention.cache_attention(q, k[:2, :, :0], v[:2, :, :0], 0).any()
    assert none.numel() == 0


def test_a_table_without_entries_is_refused():
    q, k, v, table = make([48, 48], 1, 4, 2, 128, 16)
    with pytest.raises(ValueError, match="table"):
        call(q, k[:2], v[:2], [48, 48], table[:, :0])


def test_lengths_past_the_cache_are_cut():
    q, k, v, table = make([48, 48], 1, 4, 2, 128, 16, seed=2)
    table = table[:, :3].contiguous()
    want = call(q, k, v, [48, 0], table)
    assert torch.equal(call(q, k, v, [1 << 30, -5], table), want)


def test_pages_outside_the_pool_are_not_seen():
    lens = [200, 90]
    q, k, v, table = make(lens, 3, 4, 2, 128, 16, seed=3)
    seen = torch.ones(2, 200, dtype=torch.bool)
    good = table.clone()
    for b, w, bad in ((0, 0, -1), (0, 5, k.shape[0]), (0, 12, 1 << 30), (1, 3, -(1 << 31))):
        table[b, w] = bad
        seen[b, 16 * w:16 * w + 16] = False
    got = call(q, k, v, lens, table)
    ref.check_attention(got, *ref.attention(q, k, v, lens, good, seen=seen))


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("D,S", [(128, 5), (64, 40), (256, 9)])
def test_hidden_values_that_are_not_finite(bad, D, S):
    """A new token's v reaches the rows that see it and no other."""
    n, at = 150, 150 - S + 2  # the third new token's
    q, k, v, table = make([n], S, 4, 2, D, 16, seed=S)
    page, row = int(table[0, at // 16]), at % 16
    want, tol = ref.attention(q, k, v, [n], table)
    v[page, 1, row, 3:9] = bad
    got = call(q, k, v, [n], table).cpu()
    hit = torch.zeros(1, S, 4, D, dtype=torch.bool)
    hit[:, 2:, 2:, 3:9] = True
    ref.check_attention(torch.where(hit, 0, got), torch.where(hit, 0, want), tol)
    assert not torch.isfinite(got[hit]).any()


def test_hidden_keys_that_are_not_finite():
    S, n = 4, 60
    q, k, v, table = make([n], S, 4, 2, 128, 16, seed=6)
    want, tol = ref.attention(q, k, v, [n], table)
    page, row = int(table[0, 59 // 16]), 59 % 16
    k[page, 0, row] = math.nan
    got = call(q, k, v, [n], table).cpu()
    ref.check_attention(got[:, :3], want[:, :3], tol[:, :3])
    assert torch.isnan(got[:, 3, :2]).all()
    ref.check_attention(got[:, 3:, 2:], want[:, 3:, 2:], tol[:, 3:, 2:])


def test_large_scores_and_scale():
    """One key far above the rest, scores of thousands; and a negative scale."""
    lens = [777]
    q, k, v, table = make(lens, 1, 4, 2, 128, 64, seed=7)
    q = q * 40
    for scale in (1.0, -0.5, 0.0):
        got = call(q, k, v, lens, table, scale=scale)
        ref.check_attention(got, *ref.attention(q, k, v, lens, table, scale=scale))


def test_views():
    """An arena's layer, q of a packed projection, an out with gaps, a table that is a slice."""
    g = torch.Generator().manual_seed(1)
    ar = KVArena(2, 2, 2, 90, 128, torch.bfloat16, DEV)
    ar.storage.copy_(bf16_randn(*ar.storage.shape, gen=g))
    qkv = bf16_randn(2, 3, 8 + 4, 128, gen=g).to(DEV)
    q = qkv[:, :, 1:9].transpose(1, 2)
    room = torch.full((2, 3, 9, 136), 5.0, dtype=torch.bfloat16, device=DEV)
    out = room[:, :, :8, :128]
    got = attention.cache_attention(q, ar.k(1), ar.v(1), 70, out=out)
    assert got is out
    ref.check_attention(out, *ref.attention(q, ar.k(1), ar.v(1), [70] * 2))
    assert (room[:, :, 8] == 5).all() and (room[..., 128:] == 5).all()
    q, k, v, table = make([70, 20], 1, 8, 2, 64, 16, seed=3)
    wide = torch.full((2, 40), -1, dtype=torch.int32, device=DEV)
    wide[:, 7:7 + table.shape[1]] = table
    assert torch.equal(call(q, k, v, [70, 20], wide[:, 7:7 + table.shape[1]]),
                       call(q, k, v, [70, 20], table))
    odd = bf16_randn(2, 8, 1, 65, gen=g).to(DEV)[..., 1:]
    ref.check_attention(call(odd, k, v, [70, 20], table),
                        *ref.attention(odd, k, v, [70, 20], table))


def test_offsets_past_32_bits():
    """Pages more than 2^31 elements into the pool."""
    page, Hk, D = 64, 8, 128
    pages = (1 << 31) // (page * Hk * D) + 3
    k = torch.zeros(pages, Hk, page, D, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros_like(k)
    g = torch.Generator().manual_seed(2)
    ids = [0, pages - 1, pages // 2, pages - 2]
    for p in ids:
        k[p], v[p] = (bf16_randn(Hk, page, D, gen=g).to(DEV) for _ in range(2))
    table = torch.tensor([ids], dtype=torch.int32, device=DEV)
    q = bf16_randn(1, 8, 1, D, gen=g).to(DEV)
    got = attention.cache_attention(q, k, v, 250, table=table)
    ref.check_attention(got, *ref.attention(q, k, v, [250], table))
    plan = axial.AxisPlan(torch.ones(D // 2), [0] * (D // 2), device=DEV)
    x = bf16_randn(2, Hk, D, gen=g).to(DEV)
    slots = torch.tensor([pages * page - 1, 5], device=DEV)
    pos = torch.zeros(1, 2, dtype=torch.int64, device=DEV)
    axial.rotate_append(x, x, x, pos, plan, slots, k, v)
    for c in (k, v):
        assert torch.equal(c[pages - 1, :, page - 1], x[0]) and torch.equal(c[0, :, 5], x[1])


def test_results_repeat_and_streams_agree():
    lens = [900, 33, 0, 2500]
    q, k, v, table = make(lens, 1, 8, 2, 128, 16, seed=5)
    want = call(q, k, v, lens, table)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    torch.cuda.synchronize()
    for i in range(6):  # two calls at once
        with torch.cuda.stream(side[i % 2]):
            got.append(attention.cache_attention(q, k, v, n, table=table))
    torch.cuda.synchronize()
    for o in got:
        assert torch.equal(o, want)


@pytest.mark.parametrize("S", [2, 20])
def test_two_captured_calls_share_nothing(S):
    lens = [[300, 41], [64, 1111]]
    args = [make(x, S, 8, 2, 128, 16, seed=i) for i, x in enumerate(lens)]
    ns = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in lens]
    call(*args[0][:3], lens[0], args[0][3])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for (q, k, v, table), n in zip(args, ns):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(attention.cache_attention(q, k, v, n, table=table))
        graphs.append(g)
    side = [torch.cuda.Stream() for _ in graphs]
    for step in range(3):
        for n in ns:
            n.sub_(step * 3)
        torch.cuda.synchronize()
        for g, s in zip(graphs, side):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for (q, k, v, table), n, out in zip(args, ns, outs):
            eager = attention.cache_attention(q, k, v, n, table=table)
            assert torch.equal(out, eager)
            ref.check_attention(out, *ref.attention(q, k, v, n.tolist(), table))


def test_served_together():
    """A server's steps, as a user runs them: pages planned, keys rotated into them, attended to;
    requests end and begin.  Against dense caches kept beside."""
    rng = random.Random(8)
    R, W, page, Hq, Hk, D, P = 5, 20, 16, 8, 2, 128, 90
    i32 = dict(dtype=torch.int32, device=DEV)
    n, table = torch.zeros(R, **i32), torch.zeros(R, W, **i32)
    ring, cursor = torch.arange(P, **i32), torch.tensor([0, P, 0, 0], **i32)
    k_pages, v_pages = torch.full((2, P, Hk, page, D), math.nan, dtype=torch.bfloat16, device=DEV)
    inv = (1e4 ** (-torch.arange(D // 2) / (D // 2))).float()
    plan = axial.AxisPlan(inv, torch.arange(D // 2) % 3, device=DEV)
    g = torch.Generator().manual_seed(3)
    held = [(torch.zeros(Hk, 0, D, dtype=torch.bfloat16),) * 2] * R
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
        q = axial.rotate_append(q, k, v, pos, plan, t.slots, k_pages, v_pages)
        fresh = torch.tensor(new, **i32)
        got = attention.cache_attention(q.view(R, S, Hq, D).transpose(1, 2), k_pages, v_pages, n,
                                        table=table, q_len=fresh)
        k = axial.rotate(k, k, pos, plan)[0].view(R, S, Hk, D).cpu()
        v = v.view(R, S, Hk, D).cpu()
        for r in range(R):
            past = [x[:, :0] if keep[r] == 0 else x for x in held[r]]
            held[r] = tuple(torch.cat((x, y[r, :new[r]].transpose(0, 1)), 1)
                            for x, y in zip(past, (k, v)))
            m = held[r][0].shape[1]
            assert m == int(n[r])
            want, tol = ref.attention(q.view(R, S, Hq, D).transpose(1, 2)[r:r + 1],
                                      held[r][0][None], held[r][1][None], [m], q_len=[new[r]])
            ref.check_attention(got[r:r + 1], want, tol)
