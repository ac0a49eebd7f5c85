"""Attention over a cache where values are infinite or NaN: sum p v / sum p with weights that are
above 0 for every key a row sees, as in 64 bits, whatever step, wave or workgroup a key falls to."""

from __future__ import annotations

import math

import pytest
import torch

import paged_reference as ref
from test_gpu_cache_attention import DEV, call, make
from umic.kernels import attention

pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan


def rows_of(v, table, j):
    """The [Hk, D] view of key j of the one request."""
    if table is None:
        return v[0, :, j]
    page = v.shape[2]
    return v[int(table[0, j // page]), :, j % page]


def expected(q, k, v, n, table, causal=True, scale=None):
    """The finite part and its bound (the oracle's, with the values that are not finite taken
    out), and what they make of the columns they reach: their sum."""
    fine = torch.where(torch.isfinite(v), v, 0)
    want, tol = ref.attention(q, k, fine, [n], table, causal=causal, scale=scale)
    S, Hq, Hk = q.shape[2], q.shape[1], k.shape[1]
    rows = ref.dense(v, table, 0, n).double().cpu()
    wild = torch.where(torch.isfinite(rows), 0, rows)
    for s in range(S):
        m = min(n, n - S + s + 1) if causal else n
        hit = wild[:, :m].sum(1).repeat_interleave(Hq // Hk, 0)
        want[0, s] = torch.where(hit != 0, hit, want[0, s])
    return want, tol


def check(got, want, tol):
    got = got.double().cpu()
    fine = torch.isfinite(want)
    assert not fine.all()
    assert torch.equal(got[~fine].nan_to_num(7.0, 8.0, 9.0), want[~fine].nan_to_num(7.0, 8.0, 9.0))
    ref.check_attention(torch.where(fine, got, 0), torch.where(fine, want, 0),
                        torch.where(fine, tol, 1))


def plant(q, k, v, n, table, scale=None):
    """Values that are not finite at the first key, in the middle, at the key of row 0's largest
    weight and at the last; two signs in one column, NaN in one."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    x = (ref.dense(k, table, 0, n)[0].double() @ q[0, 0, -1].double()) * scale
    top = int(x.argmax())
    for j, col, bad in ((0, 1, INF), (n // 2, 2, -INF), (n // 3, 3, INF), (top, 5, INF), (top, 6, -INF),
                        (n - 1, 8, INF), (n // 2, 9, NAN), (0, 12, INF), (n // 2, 12, -INF),
                        (n // 4, 17, -INF), (n // 5, 31, INF), (n - 1, 62, -INF)):
        rows_of(v, table, j)[-1, col] = bad


CASES = [(1, 1, 4, 2, 128, 16), (2, 1, 4, 4, 64, 0), (300, 1, 4, 2, 128, 16), (5000, 1, 4, 1, 256, 0),
         (20000, 1, 8, 2, 128, 64), (777, 1, 14, 2, 64, 32), (600, 4, 8, 2, 128, 0),
         (700, 40, 4, 2, 128, 64), (2900, 80, 8, 2, 128, 64), (900, 40, 4, 2, 256, 16),
         (500, 70, 2, 2, 64, 0)]


@pytest.mark.parametrize("n,S,Hq,Hk,D,page", CASES)
@pytest.mark.parametrize("causal", [True, False])
def test_values_that_are_not_finite(n, S, Hq, Hk, D, page, causal):
    q, k, v, table = make([n], S, Hq, Hk, D, page, seed=n + S)
    plant(q, k, v, n, table)
    want, tol = expected(q, k, v, n, table, causal)
    if causal and S == 1:  # the weights are above 0 in 64 bits too: the same from them
        rows, keys = (ref.dense(c, table, 0, n).double().cpu() for c in (v, k))
        for h in range(Hq):
            g = h // (Hq // Hk)
            p = torch.softmax(keys[g] @ q[0, h, 0].double().cpu() * D ** -0.5, 0)
            assert (p > 0).all()
            direct = (p[:, None] * rows[g]).sum(0)
            same = (direct == want[0, 0, h]) | (direct.isnan() & want[0, 0, h].isnan())
            assert (same | torch.isfinite(want[0, 0, h])).all()
    got = call(q, k, v, [n], table, causal=causal)
    check(got, want, tol)
    assert torch.equal(got.nan_to_num(7.0), call(q, k, v, [n], table, causal=causal).nan_to_num(7.0))


@pytest.mark.parametrize("n,S,Hq,Hk,D,page", [c for c in CASES if c[0] > 1])
def test_weights_that_underflow(n, S, Hq, Hk, D, page):
    """Scores of thousands: most weights are 0 in 32 bits, and the running sums are rescaled by
    factors that are."""
    q, k, v, table = make([n], S, Hq, Hk, D, page, seed=n)
    q = q * 40
    plant(q, k, v, n, table, 1.0)
    want, tol = expected(q, k, v, n, table, scale=1.0)
    check(call(q, k, v, [n], table, scale=1.0), want, tol)


@pytest.mark.parametrize("n,S", [(700, 1), (3100, 2), (900, 40)])
def test_captured(n, S):
    """The two-launch form."""
    q, k, v, table = make([n], S, 8, 2, 128, 16, seed=n)
    plant(q, k, v, n, table)
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    eager = attention.cache_attention(q, k, v, lens, table=table)
    check(eager, *expected(q, k, v, n, table))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = attention.cache_attention(q, k, v, lens, table=table)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.nan_to_num(7.0, 8.0, 9.0), eager.nan_to_num(7.0, 8.0, 9.0))


@pytest.mark.parametrize("S,Hq,Hk,D", [(2, 32, 1, 128), (5, 32, 1, 128), (3, 16, 1, 64), (2, 48, 3, 256)])
@pytest.mark.parametrize("bad", [INF, NAN])
def test_hidden_where_a_wave_has_one_token(S, Hq, Hk, D, bad):
    """Sixteen query heads and more a key head: all rows of a wave see the same keys, and not the
    later new tokens' values."""
    n = 150
    q, k, v, table = make([n], S, Hq, Hk, D, 16, seed=S)
    rows_of(v, table, n - 1)[0, 3:9] = bad
    got = call(q, k, v, [n], table)
    assert torch.isfinite(got[0, :S - 1]).all()
    check(got, *expected(q, k, v, n, table))


@pytest.mark.parametrize("S,Hq,Hk,D", [(5, 4, 4, 64), (4, 8, 2, 128), (40, 8, 2, 128), (20, 4, 2, 256)])
def test_padded_rows_and_queries_that_are_not_finite(S, Hq, Hk, D):
    """Rows past q_len are zero whatever their queries and the values hold; a NaN query's row is NaN
    and the rows beside it are not."""
    lens, fresh = [900, 2500, 70], [S - 2, 1, S]
    q, k, v, table = make(lens, S, Hq, Hk, D, 16, seed=S)
    m = torch.tensor(fresh, dtype=torch.int32, device=DEV)
    want, tol = ref.attention(q, k, v, lens, table, q_len=fresh)
    wild = q.clone()
    wild[0, :, S - 2:], wild[1, :, 1:] = NAN, INF
    wild[2, 1, S - 1] = NAN
    got = call(wild, k, v, lens, table, q_len=m)
    assert not got[0, S - 2:].any() and not got[1, 1:].any()
    assert torch.isnan(got[2, S - 1, 1]).all()
    got[2, S - 1, 1] = 0
    want[2, S - 1, 1], tol[2, S - 1, 1] = 0, 1
    ref.check_attention(got, want, tol)
