"""Calls of the 8-bit cache's operators at their edges: nothing to do, more requests than a launch
takes, streams that write beside each other, pages that two tables name."""

from __future__ import annotations

import pytest
import torch

import cache8_reference as ref8
import paged_reference as ref
from helpers import bf16_randn
from test_gpu_cache8 import DEV, KINDS, append, call, check_cache, filled, new_cache, queries, slots_of
from umic.kernels import attention, axial, cache8

pytestmark = pytest.mark.gpu


def test_nothing_to_do():
    cache = new_cache("int8", 3, 2, 16, 64)
    none = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device=DEV)
    at = torch.zeros(0, dtype=torch.int64, device=DEV)
    plan = axial.AxisPlan(torch.ones(32), [0] * 32, device=DEV)
    cache8.append(none, none, at, cache)
    q = cache8.rotate_append(none, none, none, at[None], plan, at, cache)
    assert q.shape == (0, 2, 64)
    table = torch.zeros(0, 2, dtype=torch.int32, device=DEV)
    n = torch.zeros(0, dtype=torch.int32, device=DEV)
    assert cache8.read(cache, table, n, 5)[0].shape == (0, 2, 5, 64)
    assert cache8.attention(none.view(0, 2, 0, 64), cache, n, table).shape == (0, 0, 2, 64)
    assert (cache.k.view(torch.uint8) == 0x7F).all() and (cache.k_scale == 4).all()
    # a pool without pages holds no key, and takes none
    empty = cache8.empty(0, 2, 16, 64, torch.int8, DEV)
    x = bf16_randn(3, 2, 64, gen=torch.Generator().manual_seed(1)).to(DEV)
    cache8.append(x, x, torch.arange(3, device=DEV), empty)
    table = torch.zeros(3, 2, dtype=torch.int32, device=DEV)
    n = torch.tensor([5, 0, 32], dtype=torch.int32, device=DEV)
    assert not any(t.any() for t in cache8.read(empty, table, n, 7))
    assert not cache8.attention(x.view(3, 2, 1, 64), empty, n, table).any()


@pytest.mark.parametrize("S", [1, 12])
def test_more_requests_than_a_launch_takes(S, monkeypatch):
    lens = [200, 0, 33, 17, 600, 1, 90]
    cache, table, k, v = filled("e4m3", lens, 2, 64, 16, seed=1)
    q = queries(7, S, 8, 64, 1)
    new = [S, 0, 1, S, S, 1, S]
    fresh = torch.tensor(new, dtype=torch.int32, device=DEV)
    monkeypatch.setattr(attention, "max_requests", lambda *a: 3)
    got = call(q, cache, lens, table, q_len=fresh)
    ref.check_attention(got, *ref.attention(q, k, v, lens, table.cpu(), q_len=new))
    # rows that no token was written to read as NaN, in both
    torch.testing.assert_close(
        cache8.attention(q, cache, 30, table.clamp(min=0)),
        cache8.attention(q[:, :], cache, torch.full((7,), 30, dtype=torch.int32, device=DEV),
                         table.clamp(min=0)), rtol=0, atol=0, equal_nan=True)
    monkeypatch.setattr(attention, "max_requests", lambda *a: 0)
    with pytest.raises(ValueError, match="too many"):
        call(q, cache, lens, table)


@pytest.mark.parametrize("kind", KINDS)
def test_streams_that_write_beside_each_other(kind):
    """Two requests of one pool, each on its own stream, time after time."""
    g = torch.Generator().manual_seed(3)
    page, Hk, D = 32, 4, 128
    cache = new_cache(kind, 20, Hk, page, D)
    model = list(ref8.numbers(cache))
    ids = torch.randperm(20, generator=g).view(2, 10)
    x = [[bf16_randn(n, Hk, D, scale=1.0 + i, gen=g) for n in (100, 1, 1, 40, 1)] for i in range(2)]
    where = [[], []]
    for r in range(2):
        held = 0
        for t in x[r]:
            where[r].append(slots_of(ids[r], page, held, len(t)))
            held += len(t)
    on = [[t.to(DEV) for t in y] for y in x]
    at = [[torch.tensor(s, device=DEV) for s in w] for w in where]
    side = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for step in range(5):
        for r in range(2):
            with torch.cuda.stream(side[r]):
                cache8.append(on[r][step], on[r][step], at[r][step], cache)
    torch.cuda.synchronize()
    for r in range(2):
        for t, s in zip(x[r], where[r]):
            for i in (0, 1):
                ref8.store(kind, model[i], model[i + 2], t.double().numpy(), s)
    check_cache(cache, model)


def test_pages_that_two_tables_name():
    """A prompt that requests share: read and attended to by all of them."""
    cache, table, k, v = filled("int8", [64, 30], 2, 128, 16, seed=6)
    both = table[:1].expand(3, -1).clone()
    both[1, 3:] = table[1, :both.shape[1] - 3]
    lens = [64, 48 + 16, 50]
    q = queries(3, 1, 8, 128, 6)
    got = call(q, cache, lens, both)
    ref.check_attention(got, *ref.attention(q, k, v, lens, both.cpu()))
    rows = cache8.read(cache, both, torch.tensor(lens, dtype=torch.int32, device=DEV), 64)[0].double().cpu()
    assert torch.equal(rows[1], ref.dense(k, both.cpu(), 1, 64)) and torch.equal(rows[0, :, :48], rows[1, :, :48])


def test_e4m3_codes_from_elsewhere():
    """Scales and codes that another program made: subnormal codes, the largest ones, -0."""
    g = torch.Generator().manual_seed(8)
    bits = torch.randint(0, 256, (2, 6, 2, 16, 64), generator=g, dtype=torch.uint8)
    bits[(bits & 0x7F) == 0x7F] = 0x7E  # not the NaNs
    scale = torch.exp2(torch.randint(-20, 9, (2, 6, 2, 1), generator=g).float())
    cache = cache8.Pages8(*bits.to(DEV).view(torch.float8_e4m3fn), *scale.to(DEV))
    values = bits.view(torch.float8_e4m3fn).double() * scale.double()[..., None]
    table = torch.tensor([[3, 1, 0], [2, 5, 4]], dtype=torch.int32, device=DEV)
    got = cache8.read(cache, table, 48, 48)
    for x, y in zip(got, values):
        for b in range(2):
            assert torch.equal(x[b].double().cpu(), ref.dense(y, table.cpu(), b, 48))
    for S in (1, 20):
        q = queries(2, S, 4, 64, S) * 2.0 ** -12
        got = cache8.attention(q, cache, 48, table)
        ref.check_attention(got, *ref.attention(q, *values, [48] * 2, table.cpu()))


def test_refusals_of_shapes_and_types():
    cache = new_cache("int8", 3, 2, 16, 64)
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device=DEV)
    at = torch.arange(4, device=DEV)
    table = torch.zeros(4, 2, dtype=torch.int32, device=DEV)
    n = torch.ones(4, dtype=torch.int32, device=DEV)
    for bad in ((x[:, :1], x[:, :1], at), (x[..., :32], x[..., :32], at), (x, x[:3], at), (x, x, at[:3]),
                (x, x, at.int()), (x, x, at.repeat_interleave(2)[::2])):
        with pytest.raises(ValueError):
            cache8.append(*bad, cache)
    with pytest.raises(TypeError):
        cache8.append(x.float(), x.float(), at, cache)
    with pytest.raises(ValueError, match="cache is on"):
        cache8.append(x, x, at, cache8.empty(3, 2, 16, 64, torch.int8, "cpu"))
    grad = x.clone().requires_grad_()
    for call_ in (lambda: cache8.append(grad, x, at, cache), lambda: cache8.append(x, grad, at, cache),
                  lambda: cache8.attention(grad[:, :, None], cache, n, table)):
        with pytest.raises(RuntimeError, match="no backward"):
            call_()
    q = x[:, :, None]
    for kw in (dict(kv_len=33), dict(kv_len=n.long()), dict(kv_len=n[:3]), dict(table=table[:3]),
               dict(table=table.long()), dict(q=q[..., :32]), dict(q=q[:, :1]), dict(q_len=n[:2]),
               dict(out=torch.zeros(4, 2, 1, 64, dtype=torch.bfloat16, device=DEV))):
        args = dict(q=q, cache=cache, kv_len=n, table=table) | kw
        with pytest.raises(ValueError):
            cache8.attention(**args)
    for kw in (dict(kv_len=33), dict(rows=-1), dict(start=n.long()), dict(table=table[0])):
        with pytest.raises(ValueError):
            cache8.read(**(dict(cache=cache, table=table, kv_len=n, rows=3) | kw))
    assert (cache.k.view(torch.uint8) == 0x7F).all()
