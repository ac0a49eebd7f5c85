"""Page plans (umic_page_plan) against a request-by-request form on the host: the same
lengths, queue, table entries, slots and positions, whole numbers equal."""

from __future__ import annotations

import random

import numpy as np
import pytest
import torch

import paged_reference as ref
from umic.kernels import paged

pytestmark = pytest.mark.gpu


def state(rng, R, W, page, spare):
    """Requests of random lengths over a shuffled pool with `spare` free pages."""
    lens = [rng.choice((0, 1, page, page + 1, rng.randint(0, W * page))) for _ in range(R)]
    lens = [min(n, W * page) for n in lens]
    have = [-(-n // page) for n in lens]
    ids = np.random.RandomState(rng.randint(0, 1 << 30)).permutation(sum(have) + spare)
    table = np.full((R, W), -7, np.int32)
    at = 0
    for r, c in enumerate(have):
        table[r, :c] = ids[at:at + c]
        at += c
    ring = np.full(len(ids), -9, np.int32)
    head = rng.randrange(len(ids)) if len(ids) else 0
    for i in range(spare):
        ring[(head + i) % len(ids)] = ids[at + i]
    return np.array(lens, np.int32), table, ring, np.array([head, spare, 5, 5], np.int32)


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()


def run(lens, new, table, ring, cursor, page, tokens, keep=None, delta=None, row=0, out=None):
    t, g = dev(table), dev(ring)
    step = paged.plan_pages(dev(lens), dev(new), t, g, dev(cursor), page, tokens,
                            keep=None if keep is None else dev(keep),
                            delta=None if delta is None else dev(delta), row=row, out=out)
    return [x.cpu().numpy() for x in (*step, t, g)]


def check(got, want):
    for name, a, b in zip(("kv_len", "cursor", "starts", "slots", "positions", "table", "ring"),
                          got, want):
        assert a.dtype == b.dtype and np.array_equal(a, b), (name, a, b)


@pytest.mark.parametrize("R", [1, 7, 64, 257, 1025, 2300])
@pytest.mark.parametrize("page", [16, 64])
def test_steps(R, page):
    rng = random.Random(R * 100 + page)
    W = 9 if R > 300 else 33
    lens, table, ring, cursor = state(rng, R, W, page, 8 * R)
    keep = [rng.choice((-3, 0, 1, rng.randint(0, 40), 1 << 30)) for _ in lens]
    new = [rng.choice((-1, 0, 1, page, rng.randint(0, 3 * page))) for _ in lens]
    new = [min(x, W * page - min(max(k, 0), int(n))) for x, k, n in zip(new, keep, lens)]
    delta = [rng.randint(-900, 900) for _ in lens]
    total = sum(max(x, 0) for x in new)
    for k, d, spare in ((keep, delta, 0), (None, None, 13)):
        fresh = new if k is not None else [min(x, W * page - int(n)) for x, n in zip(new, lens)]
        args = (lens, fresh, table, ring, cursor, page, total + spare, k, d)
        want = ref.plan(*args)
        assert want[1][3] in (0, 1)
        check(run(*args), want)


@pytest.mark.parametrize("row", [1, 5, 130])
def test_padded_rows(row):
    rng = random.Random(row)
    lens, table, ring, cursor = state(rng, 37, 24, 32, 300)
    lens = np.minimum(lens, 24 * 32 - row).astype(np.int32)
    new = [rng.randint(0, row) for _ in lens]
    keep = [int(n) for n in lens]
    args = (lens, new, table, ring, cursor, 32, 37 * row, keep, None, row)
    want = ref.plan(*args)
    assert want[1][3] == paged.PLAN_OK
    check(run(*args), want)


@pytest.mark.parametrize("why", ["pages", "long", "room", "row", "negative", "wide", "head", "count",
                                 "full"])
def test_refused_steps_change_nothing(why):
    page, W = 16, 4
    lens = np.array([20, 0, 64], np.int32)
    table = np.array([[5, 6, -1, -1], [-1] * 4, [0, 1, 2, 3]], np.int32)
    ring = np.array([4, 7, 8, -1, -1, -1, -1, -1, -1], np.int32)
    cursor = np.array([0, 3, 0, 0], np.int32)
    new, keep, tokens, row = [1, 1, 0], None, 8, 0
    status = paged.NO_PAGES
    if why == "pages":
        new = [44, 33, 0]      # 2 + 3 pages, 3 free
        tokens = 100
    elif why == "long":
        new, status = [45, 0, 0], paged.TOO_LONG
        tokens = 100
    elif why == "room":
        new, status = [5, 4, 0], paged.NO_ROOM
    elif why == "row":
        new, tokens, row, status = [3, 1, 0], 6, 2, paged.NO_ROOM
    elif why == "negative":
        lens[1], status = -1, paged.BAD_STATE
    elif why == "wide":
        lens[2], status = 65, paged.BAD_STATE
    elif why == "head":
        cursor[0], status = 9, paged.BAD_STATE
    elif why == "count":
        cursor[1], status = -1, paged.BAD_STATE
    else:
        keep, cursor[1], status = [20, 0, 0], 6, paged.BAD_STATE  # 4 come back to 6 of 9
    args = (lens, new, table, ring, cursor, page, tokens, keep, None, row)
    want = ref.plan(*args)
    assert want[1][3] == status
    check(run(*args), want)


def test_lengths_end_at_32_bits():
    page, most = 1 << 30, (1 << 31) - 1
    table, ring = np.array([[2, 1, -1]], np.int32), np.array([0, -1, -1], np.int32)
    for new, want in ((4, paged.PLAN_OK), (5, paged.TOO_LONG)):
        got = run(np.array([most - 4], np.int32), [new], table, ring,
                  np.array([0, 1, 0, 0], np.int32), page, 8, None, None, 0)
        assert got[1][3] == want
        assert got[0][0] == (most if want == paged.PLAN_OK else most - 4)
        assert got[3][0] == ((1 << 30) + (most - 4) % page if want == paged.PLAN_OK else -1)


def test_in_place_and_repeated():
    """kv_len and cursor as their own outputs; and a step repeated on the same lengths and queue."""
    rng = random.Random(3)
    lens, table, ring, cursor = state(rng, 20, 16, 16, 100)
    keep = [int(n) // 2 for n in lens]
    new = [min(9, 16 * 16 - k) for k in keep]
    want = ref.plan(lens, new, table, ring, cursor, 16, 200, keep)
    t, g, n, c = dev(table), dev(ring), dev(lens), dev(cursor)
    for _ in range(3):
        step = paged.plan_pages(n, dev(new), t, g, c, 16, 200, keep=dev(keep))
        check([x.cpu().numpy() for x in (*step, t, g)], want)
    own = paged.PageStep(n, c, *step[2:])
    step = paged.plan_pages(n, dev(new), t, g, c, 16, 200, keep=dev(keep), out=own)
    assert step.kv_len is n and step.cursor is c
    check([x.cpu().numpy() for x in (*step, t, g)], want)


def test_a_long_run_keeps_every_page_once():
    """Steps of a server: requests end, begin and go on; a page is never in two places."""
    rng = random.Random(11)
    R, W, page, P = 24, 20, 16, 300
    lens, table = np.zeros(R, np.int32), np.full((R, W), -1, np.int32)
    ring, cursor = np.arange(P, dtype=np.int32), np.array([0, P, 0, 0], np.int32)
    n, t, g, c = dev(lens), dev(table), dev(ring), dev(cursor)
    for _ in range(40):
        keep = [0 if rng.random() < 0.2 else 1 << 30 for _ in range(R)]
        new = [rng.randint(1, 90) if k == 0 or x == 0 else 1 for k, x in zip(keep, lens)]
        new = [min(x, W * page - (int(m) if k else 0)) for x, k, m in zip(new, keep, lens)]
        want = ref.plan(lens, new, table, ring, cursor, page, R * 90, keep)
        own = paged.PageStep(n, c, *(torch.empty_like(x) for x in paged.plan_pages(
            n, dev(new), t.clone(), g.clone(), c, page, R * 90, keep=dev(keep))[2:]))
        step = paged.plan_pages(n, dev(new), t, g, c, page, R * 90, keep=dev(keep), out=own)
        check([x.cpu().numpy() for x in (*step, t, g)], want)
        lens, cursor, _, slots, _, table, ring = want
        held = [p for r in range(R) for p in table[r, :-(-int(lens[r]) // page)]]
        queue = [ring[(cursor[0] + i) % P] for i in range(cursor[1])]
        assert sorted(held + queue) == list(range(P))
        real = slots[slots >= 0]
        assert len(set(real.tolist())) == len(real)


def test_captured_step_replays():
    """One graph of a step, replayed: lengths and queue go on from replay to replay."""
    R, page, W = 6, 16, 8
    lens, cursor = np.array([3, 0, 15, 16, 31, 32], np.int32), np.array([7, 30, 0, 0], np.int32)
    table = np.full((R, W), -1, np.int32)
    at = 30
    for r, m in enumerate(lens):
        for w in range(-(-int(m) // page)):
            table[r, w] = at
            at += 1
    ring = np.full(at, -1, np.int32)
    for i in range(30):
        ring[(7 + i) % at] = i
    new = np.ones(R, np.int32)
    n, t, g, c, f = dev(lens), dev(table), dev(ring), dev(cursor), dev(new)
    out = paged.PageStep(n, c, *(x.clone() for x in paged.plan_pages(n, f, t.clone(), g.clone(), c,
                                                                     page, R)[2:]))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.plan_pages(n, f, t, g, c, page, R, out=out)
    for i in range(20):
        want = ref.plan(lens, new, table, ring, cursor, page, R)
        graph.replay()
        torch.cuda.synchronize()
        check([x.cpu().numpy() for x in (*out, t, g)], want)
        lens, cursor, table, ring = want[0], want[1], want[5], want[6]
        assert f.sum().item() == R  # eager work between the replays


def test_no_requests():
    z = torch.zeros(0, dtype=torch.int32, device="cuda")
    c = dev([2, 5, 9, 9])
    step = paged.plan_pages(z, z, z.view(0, 3), dev(np.arange(8)), c, 16, 0)
    assert step.cursor.tolist() == [2, 5, 0, 0] and step.starts.tolist() == [0]
