"""A paged cache whose steps were replayed from a graph, and steps that the device refuses."""

from __future__ import annotations

import pytest
import torch

import paged_reference as ref
from helpers import bf16_randn, rel_err
from test_gpu_cache_attention import make
from test_gpu_paged_cache import TOL, text_model
from umic.kernels import attention, paged
from umic.paged_cache import PagedArena, PagedKVCache

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore::FutureWarning"),
              pytest.mark.filterwarnings("ignore::UserWarning")]
DEV = "cuda"


def arena(requests=3, pages=12):
    return PagedArena(1, requests, pages, 2, 16, 64, 64)


def replayed(ar, steps):
    """Steps of one token each past ``ar.plan``, as a captured plan makes them."""
    fresh = torch.ones(ar.requests, dtype=torch.int32, device=DEV)
    slots, positions = torch.empty(2, ar.requests, dtype=torch.int64, device=DEV)
    out = paged.PageStep(ar.kv_len, ar.cursor, fresh.new_empty(ar.requests + 1), slots, positions)
    for _ in range(steps):
        paged.plan_pages(ar.kv_len, fresh, ar.table, ar.ring, ar.cursor, 16, ar.requests, row=1,
                         out=out)


def test_what_is_kept_is_the_devices():
    """None keeps all that a request holds on the device, and a number at most that."""
    ar = arena()
    ar.plan([20, 5, 13])
    replayed(ar, 14)
    assert ar.kv_len.tolist() == [34, 19, 27] and ar.lens == [20, 5, 13]
    ar.plan([1, 1, 1], keep=[0, None, 25])
    assert ar.kv_len.tolist() == [1, 20, 26]
    ar.sync()
    assert ar.lens == [1, 20, 26] and ar.free == 12 - 1 - 2 - 2 == ar.cursor.tolist()[1]


def test_sync_says_what_was_refused():
    ar = arena(pages=4)
    ar.plan([20, 5, 13])
    replayed(ar, 13)  # the third request would need a second page and a third
    assert ar.kv_len.tolist() != ar.lens
    with pytest.raises(RuntimeError, match="pages are missing"):
        ar.sync()
    assert ar.lens == ar.kv_len.tolist() and ar.free == ar.cursor.tolist()[1]
    ar.plan([1, 0, 0], keep=[0, 0, 0])
    ar.sync()
    assert ar.lens == [1, 0, 0] and ar.free == 3


def test_a_request_starts_anew_after_replays():
    """A captured decode step's replays, then a step in which one request starts anew: the others'
    tokens stay."""
    m, _ = text_model()
    g = torch.Generator().manual_seed(4)
    prompt = torch.randint(0, 512, (3, 20), generator=g).to(DEV)
    ids = torch.zeros(3, 1, dtype=torch.long, device=DEV)
    caches = []
    with torch.no_grad():
        for _ in range(2):
            c = PagedKVCache.for_model(m, requests=3, pages=12, max_tokens=64, page_size=16)
            for new, tokens in (([20, 5, 13], prompt), (1, ids)):
                c.begin(new)
                m(input_ids=tokens, position_ids=c.position_ids, past_key_values=c)
            caches.append(c)
        graphed, eager = caches
        ar = graphed.arena
        fresh = torch.ones(3, dtype=torch.int32, device=DEV)
        out = graphed.step = paged.PageStep(ar.kv_len, ar.cursor, *graphed.step[2:])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            paged.plan_pages(ar.kv_len, fresh, ar.table, ar.ring, ar.cursor, 16, 3, row=1, out=out)
            graphed._positions = out.positions.expand(3, -1)
            m(input_ids=ids, position_ids=graphed.position_ids, past_key_values=graphed)
        for _ in range(15):
            ids.copy_(torch.randint(0, 512, (3, 1), generator=g))
            eager.begin(1)
            m(input_ids=ids, position_ids=eager.position_ids, past_key_values=eager)
            graph.replay()
        graphed.sync()
        assert ar.lens == eager.arena.lens == [36, 21, 29] and ar.free == eager.arena.free
        for keep in ([0, None, None], [None, 7, None], None):
            outs = []
            for c in caches:
                c.begin(1, keep=keep)
                outs.append(m(input_ids=ids, position_ids=c.position_ids,
                              past_key_values=c).last_hidden_state)
            assert torch.equal(*outs)
            assert ar.kv_len.tolist() == eager.arena.kv_len.tolist() == ar.lens
            assert ar.cursor.tolist()[1::2] == [ar.free, 0]


def test_replays_and_plans_in_turn():
    """Steps replayed from a graph and steps planned between them: one set of lengths and pages."""
    ar, other = arena(requests=4, pages=14), arena(requests=4, pages=14)
    for a in (ar, other):
        a.plan([20, 5, 13, 1])
    fresh = torch.ones(4, dtype=torch.int32, device=DEV)
    slots, positions = torch.empty(2, 4, dtype=torch.int64, device=DEV)
    out = paged.PageStep(ar.kv_len, ar.cursor, fresh.new_empty(5), slots, positions)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.plan_pages(ar.kv_len, fresh, ar.table, ar.ring, ar.cursor, 16, 4, row=1, out=out)
    for keep in ([None, 0, None, None], [30, None, None, 2], [0, 0, None, None]):
        for _ in range(9):
            graph.replay()
            want, _ = other.plan([1] * 4)
            assert torch.equal(slots, want.slots) and torch.equal(positions, want.positions)
        ar.sync()
        new = [17, 2, 1, 0]
        for got, want in zip(*(a.plan(new, keep)[0] for a in (ar, other))):
            assert torch.equal(got, want)
        for a in (ar, other):
            assert a.kv_len.tolist() == a.lens and a.cursor.tolist()[1::2] == [a.free, 0]
        # no page twice
        held = [p for r, n in enumerate(ar.lens) for p in ar.table[r, :-(-n // 16)].tolist()]
        assert len(set(held)) == len(held) == 14 - ar.free


@pytest.mark.parametrize("given", [False, True])
def test_no_requests_and_entries(given):
    """Every entry says that there is no token, also in the caller's tensors."""
    i32 = dict(dtype=torch.int32, device=DEV)
    none, table = torch.empty(0, **i32), torch.empty(0, 3, **i32)
    ring, cursor = torch.arange(4, **i32), torch.tensor([1, 3, 9, 9], **i32)
    out = None
    if given:
        longs = torch.full((2, 7), 5, dtype=torch.int64, device=DEV)
        out = paged.PageStep(none, torch.full((4,), 5, **i32), torch.full((1,), 5, **i32), *longs)
    else:  # what torch.empty is likely to give
        torch.full((2, 7), 5, dtype=torch.int64, device=DEV)
    step = paged.plan_pages(none, none, table, ring, cursor, 16, 7, out=out)
    assert step.slots.tolist() == [-1] * 7 and step.positions.tolist() == [0] * 7
    assert step.cursor.tolist() == [1, 3, 0, 0] and step.starts.tolist() == [0]


@pytest.mark.parametrize("S", [1, 3, 40])
@pytest.mark.parametrize("own_out", [False, True])
def test_more_requests_than_one_launch_takes(S, own_out):
    """A table of 2^30 tokens a request: 63 requests a launch."""
    B, W, page, Hq, D = 70, 1 << 14, 1 << 16, 2, 64
    assert attention.max_requests(S, Hq, 1, D, W * page) == 63
    g = torch.Generator().manual_seed(S)
    k, v = (bf16_randn(3, 1, page, D, gen=g).to(DEV) for _ in range(2))
    q = bf16_randn(B, S, Hq, D, scale=1.5, gen=g).to(DEV).transpose(1, 2)
    table = torch.full((B, W), -1, dtype=torch.int32, device=DEV)
    table[:, 0], table[:, 1] = torch.arange(B) % 3, torch.arange(1, B + 1) % 3
    lens = [(b * b * 13) % 300 for b in range(B)]
    lens[5], lens[62], lens[63], lens[69] = page + 100, 0, page + 7, 301
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    fresh = [min(S, b % (S + 1)) for b in range(B)]
    m = torch.tensor(fresh, dtype=torch.int32, device=DEV)
    out = torch.full((B, S, Hq, D), 7.0, dtype=torch.bfloat16, device=DEV) if own_out else None
    got = attention.cache_attention(q, k, v, n, table=table, q_len=m, out=out)
    assert out is None or got is out
    ref.check_attention(got, *ref.attention(q, k, v, lens, table, q_len=fresh))
    for b in (62, 63):
        part = slice(b, b + 1)
        alone = attention.cache_attention(q[part], k, v, n[part], table=table[part, :4], q_len=m[part])
        ref.check_attention(alone, *ref.attention(q[part], k, v, lens[part], table[part],
                                                  q_len=fresh[part]))
    same = attention.cache_attention(q, k, v, 200, table=table, causal=False)
    ref.check_attention(same, *ref.attention(q, k, v, [200] * B, table, causal=False))


@pytest.mark.parametrize("page", [0, 16])
def test_requests_of_several_launches(monkeypatch, page):
    """Contiguous caches and tables, cut into launches of three requests."""
    lens, S = [40, 0, 200, 33, 7, 90, 150], 5
    q, k, v, table = make(lens, S, 8, 2, 128, page, seed=page)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    m = torch.tensor([5, 0, 3, 5, 5, 1, 2], dtype=torch.int32, device=DEV)
    monkeypatch.setattr(attention, "max_requests", lambda *a: 3)
    got = attention.cache_attention(q, k, v, n, table=table, q_len=m)
    ref.check_attention(got, *ref.attention(q, k, v, lens, table, q_len=m.tolist()))
    if not page:
        k, v = k.nan_to_num(0.5), v.nan_to_num(0.5)
        got = attention.cache_attention(q, k, v, 100)
        ref.check_attention(got, *ref.attention(q, k, v, [100] * 7))
    monkeypatch.setattr(attention, "max_requests", lambda *a: 0)
    with pytest.raises(ValueError, match="one launch"):
        attention.cache_attention(q, k, v, n, table=table)


def test_positions_of_the_forward():
    """The forward's position ids are the step's, or refused: its attention turns by the step's."""
    m, _ = text_model()
    c = PagedKVCache.for_model(m, requests=2, pages=12, max_tokens=64, page_size=16)
    g = torch.Generator().manual_seed(7)
    ids = torch.randint(0, 512, (2, 9), generator=g).to(DEV)

    def run(pos, *where):
        c.reset()
        c.begin([9, 4], *where)
        return m(input_ids=ids, position_ids=pos, past_key_values=c).last_hidden_state

    with torch.no_grad():
        c.begin([9, 4])
        own = c.position_ids.clone()
        image = torch.randint(0, 30, (3, 2, 9), generator=g).to(DEV)
        padded = own.clone()
        padded[:, 1, 4:] = 17  # rows without a token
        text = torch.cat((own[:1] + 3, own))
        want = run(None)
        for pos in (own, own[0], own[:1], padded, text):
            assert torch.equal(run(pos)[0], want[0]) and torch.equal(run(pos)[1, :4], want[1, :4])
        for pos in (image, own + 1, image[0], torch.cat((own, image))[:5], own.cpu()):
            with pytest.raises(ValueError, match="position_ids"):
                run(pos)
        got = run(image, image)
        assert not torch.equal(got[0], want[0])
        c.reset()
        c.begin([9, 4], image)
        assert torch.equal(m(input_ids=ids, position_ids=c.position_ids,
                             past_key_values=c).last_hidden_state[0], got[0])
        with pytest.raises(ValueError, match="position_ids"):
            run(own, image)
        with pytest.raises(ValueError, match="position_ids"):
            m(ids, None, own, c)


@pytest.mark.parametrize("how", ["module", "call", "neither"])
def test_attention_that_is_not_causal(how):
    """By the module's attribute or the call's word: every new token of a request sees the others.
    Against the unpatched module on the CPU, with a mask that shows all."""
    m, plain = text_model()
    c = PagedKVCache.for_model(m, requests=2, pages=8, max_tokens=64, page_size=16)
    g = torch.Generator().manual_seed(8)
    x = torch.randn(2, 12, 256, generator=g).to(torch.bfloat16)
    attn = m.layers[0].self_attn
    if how == "module":
        attn.is_causal = False
    lens = [12, 7]
    with torch.no_grad():
        c.begin(lens)
        got = attn(x.to(DEV), (None, None), None, past_key_values=c,
                   **({"is_causal": False} if how == "call" else {}))[0]
        for r, n in enumerate(lens):
            rot = plain.rotary_emb(x[r:r + 1], torch.arange(n).expand(3, 1, n))
            mask = torch.zeros(1, 1, n, n, dtype=torch.bfloat16)
            if how == "neither":
                mask += torch.full((n, n), float("-inf")).triu(1).to(torch.bfloat16)
            want = plain.layers[0].self_attn(x[r:r + 1, :n], rot, mask)[0]
            assert rel_err(got[r, :n], want[0]) <= TOL


def test_workspaces_of_many_streams():
    """As many are held as the module says, whatever streams have called."""
    lens = [900, 33, 0, 2500]
    q, k, v, table = make(lens, 5, 8, 2, 128, 16, seed=5)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    want = attention.cache_attention(q, k, v, n, table=table)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(7)]
    got = []
    for i in range(21):
        with torch.cuda.stream(streams[i * 3 % 7]):
            got.append(attention.cache_attention(q, k, v, n, table=table))
            if i % 2:  # single tokens, with counters
                attention.cache_attention(q[:, :, :1], k, v, n, table=table)
        assert len(attention._SCRATCH) <= attention.SCRATCH_STREAMS
    torch.cuda.synchronize()
    for o in got:
        assert torch.equal(o, want)
    for counters, _ in attention._SCRATCH.values():
        assert not counters.any()


def test_positions_that_stand_for_several_requests():
    """One row of position ids for all requests is compared with each, as are those of embeddings."""
    m, _ = text_model()
    c = PagedKVCache.for_model(m, requests=2, pages=12, max_tokens=64, page_size=16)
    ids = torch.randint(0, 512, (2, 6), generator=torch.Generator().manual_seed(9)).to(DEV)
    row = torch.arange(6, device=DEV)[None]
    with torch.no_grad():
        emb = m.embed_tokens(ids)
        for pos in (row, row[None].expand(3, 1, 6), None):
            c.reset()
            c.begin(6)
            got = m(inputs_embeds=emb, position_ids=pos, past_key_values=c).last_hidden_state
        for pos in (row + 1, row[None].expand(3, 1, 6) * 2, row[:, :3], row[:, :5], row[None, None]):
            for tokens in ({"input_ids": ids}, {"inputs_embeds": emb}):
                with pytest.raises(ValueError, match="position_ids"):
                    m(**tokens, position_ids=pos, past_key_values=c)
        c.begin([1, 1], keep=[3, None])  # requests that are not alike
        last = torch.tensor([[3]], device=DEV)
        with pytest.raises(ValueError, match="position_ids"):
            m(input_ids=ids[:, :1], position_ids=last, past_key_values=c)
        c.reset()
        c.begin(6)
        assert torch.equal(m(input_ids=ids, past_key_values=c).last_hidden_state, got)
