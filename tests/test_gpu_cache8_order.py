"""Tokens of a block that stand anywhere in a call: written once, as a whole, whatever the order of
the slots.  Codes and scales bit for bit: against the plain form in 64 bits, and against the same
tokens in order."""

from __future__ import annotations

import pytest
import torch

import cache8_reference as ref8
from helpers import bf16_randn
from test_gpu_cache8 import DEV, KINDS, append, new_cache, slots_of, spread
from umic.kernels import axial, cache8

pytestmark = pytest.mark.gpu


def in_turn(prompts, n, page):
    """Slots of prompts whose tokens alternate, each on pages of its own."""
    pages = -(-n // page)
    return [slots_of(range(r * pages, (r + 1) * pages), page, 0, n)[i] for i in range(n) for r in range(prompts)]


def far_ends(T):
    """A block's first and last row at the call's ends, its others in the middle; -1 between."""
    slots = [-1] * T
    slots[0], slots[-1] = 21, 30
    for i in range(8):
        slots[T // 2 + 3 * i] = 29 - i
    return slots


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("name", ["2 prompts of 16", "4 prompts of 16", "5 prompts of 100", "two tokens",
                                  "far ends", "far ends of many", "a block each way"])
@pytest.mark.parametrize("Hk,D,page", [(2, 64, 16), (3, 128, 32), (1, 256, 16)])
def test_orders(kind, name, Hk, D, page):
    slots = {"2 prompts of 16": lambda: in_turn(2, 16, page), "4 prompts of 16": lambda: in_turn(4, 16, page),
             "5 prompts of 100": lambda: in_turn(5, 100, page), "two tokens": lambda: [5] + [-1] * 30 + [4],
             "far ends": lambda: far_ends(70), "far ends of many": lambda: far_ends(5000),
             "a block each way": lambda: list(range(40)) + [-1] * 40 + list(range(80, 40, -1))}[name]()
    g = torch.Generator().manual_seed(len(slots) + D)
    cache = new_cache(kind, max(slots) // page + 2, Hk, page, D)
    model = list(ref8.numbers(cache))
    for step in range(2):
        k, v = (spread(g, len(slots), Hk, D) for _ in range(2))
        append(kind, cache, model, k, v, slots)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T,room", [(25, 32), (64, 80), (300, 320), (300, 4000), (2048, 2200), (2049, 2200), (5000, 5200)])
def test_shuffled(kind, T, room):
    """All slots, or some of many, in no order at all; a third of them again, behind other rows."""
    g = torch.Generator().manual_seed(T + room)
    page, Hk, D = 16, 2, 128
    cache = new_cache(kind, -(-room // page), Hk, page, D)
    model = list(ref8.numbers(cache))
    slots = torch.randperm(room, generator=g)[:T].tolist()
    k, v = (spread(g, T, Hk, D) for _ in range(2))
    append(kind, cache, model, k, v, slots)
    again = [s if i % 3 == 0 else -1 for i, s in enumerate(slots)]
    append(kind, cache, model, v, k, again)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [40, 700, 3000])
@pytest.mark.parametrize("Hq,Hk,D", [(8, 2, 128), (4, 3, 64), (4, 1, 256)])
@pytest.mark.parametrize("norm", [False, True])
def test_rotated_tokens_in_any_order(kind, T, Hq, Hk, D, norm):
    """q's rows and the cache are those of the same tokens in order."""
    g = torch.Generator().manual_seed(T + D)
    q, k, v = (bf16_randn(T, h, D, gen=g).to(DEV) for h in (Hq, Hk, Hk))
    inv, axis = (1e4 ** (-torch.arange(D // 2) / (D // 2))).float(), torch.arange(D // 2) % 3
    plan = axial.AxisPlan(inv, axis, 1.25, DEV)
    pos = torch.randint(-9, 40000, (3, T), generator=g).to(DEV)
    weights = tuple(bf16_randn(D, scale=0.1, shift=1.0, gen=g).to(DEV) for _ in range(2)) + (1e-5,)
    slots = torch.arange(T, device=DEV) + 5
    slots[::7] = -1
    one, two = (new_cache(kind, T // 16 + 2, Hk, 16, D) for _ in range(2))
    want = cache8.rotate_append(q, k, v, pos, plan, slots, one, weights if norm else None)
    order = torch.randperm(T, generator=g).to(DEV)
    got = cache8.rotate_append(q[order], k[order], v[order], pos[:, order], plan, slots[order], two,
                               weights if norm else None)
    assert torch.equal(got, want[order])
    for a, b in zip(one, two):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_captured_append_of_another_order():
    """A captured call whose slots change from replay to replay: near each other, then apart."""
    g = torch.Generator().manual_seed(9)
    T, Hk, D, page = 96, 2, 64, 16
    cache = new_cache("int8", T // page, Hk, page, D)
    k, v = (bf16_randn(T, Hk, D, gen=g) for _ in range(2))
    kd, vd, at = k.to(DEV), v.to(DEV), torch.arange(T, device=DEV)
    cache8.append(kd, vd, at, cache)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        cache8.append(kd, vd, at, cache)
    for order in (torch.arange(T), torch.randperm(T, generator=g), torch.arange(T).flip(0),
                  torch.randperm(T, generator=g)):
        at.copy_(order)
        graph.replay()
        torch.cuda.synchronize()
        model = [x * 0 for x in ref8.numbers(cache)]
        for i, x in enumerate((k, v)):
            ref8.store("int8", model[i], model[i + 2], x.double().numpy(), order.tolist())
        for got, want in zip(ref8.numbers(cache), model):
            assert (got == want).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [1, 24, 25, 63, 64, 65, 1025, 2047, 2048, 2051, 4097])
def test_any_number_of_tokens(kind, T):
    """In order with and without a lead, in turn, in no order, with gaps."""
    g = torch.Generator().manual_seed(T)
    page, Hk, D = 32, 1, 64
    room = 2 * T + 70
    order = torch.randperm(room, generator=g)[:T].tolist()
    for slots in (list(range(T)), list(range(7, T + 7)), in_turn(2, T, page)[:T], order,
                  [-1 if i % 11 == 3 else s for i, s in enumerate(range(5, T + 5))]):
        cache = new_cache(kind, -(-room // page) + 2, Hk, page, D)
        model = list(ref8.numbers(cache))
        k, v = (spread(g, T, Hk, D) for _ in range(2))
        append(kind, cache, model, k, v, slots)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("name", ["prompts", "two halves", "shuffled"])
def test_many_tokens(kind, name):
    """More chunks than the chip holds workgroups: ragged prompts, whose blocks are whole but for
    their ends; a prompt's odd rows, then its even ones; no order."""
    T, page, Hk, D = 70001, 16, 1, 64
    g = torch.Generator().manual_seed(3)
    slots, at = [], 0
    for i in range(9):
        n = T // 9 if i < 8 else T - len(slots)
        slots += range(at + 3 * i, at + 3 * i + n)
        at += n + 64 - n % 16
    if name == "two halves":
        slots = list(range(1, T, 2)) + list(range(0, T, 2))
    if name == "shuffled":
        slots = torch.randperm(T + 100, generator=g)[:T].tolist()
    slots[T // 2] = -1
    cache = new_cache(kind, max(slots) // page + 1, Hk, page, D)
    model = list(ref8.numbers(cache))
    k, v = (spread(g, T, Hk, D) for _ in range(2))
    append(kind, cache, model, k, v, slots)
    q = bf16_randn(T, 2, D, gen=g).to(DEV)
    plan = axial.AxisPlan(torch.zeros(D // 2), [0] * (D // 2), device=DEV)  # nothing turns
    twin = new_cache(kind, cache.k.shape[0], Hk, page, D)
    out = cache8.rotate_append(q, k.to(DEV), v.to(DEV), torch.zeros(1, T, dtype=torch.int64, device=DEV),
                               plan, torch.tensor(slots, device=DEV), twin)
    assert torch.equal(out, q)
    for a, b in zip(cache, twin):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
