"""The paged cache's operators as timed cases: pages planned from request lengths,
rotary positions of several axes written into the pages, and attention of new
tokens over a cache.

`own` false computes them in elementary torch operations, in 32 bits (angles in
64); `own` true makes the package's calls.  The sizes are the package's own (a
text trunk of 32 query and 8 key / value heads of 128, a vision encoder of 16
heads of 80, a prompt of about 3100 tokens, an action expert of 32 to 64 tokens
a step) and generic ones for a server of many requests.
"""

from __future__ import annotations

import functools
import math
import os
import random
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
BF = torch.bfloat16
EPS = 1e-6
THETA = {"text": 1e6, "vision": 1e4}
SECTIONS = {128: (24, 20, 20), 64: (12, 10, 10), 256: (48, 40, 40)}  # time, height, width


def listed():
    return [
        # one decode step of eight requests: one token each, now and then a new page
        {"name": "plan_decode", "op": "plan", "requests": 8, "held": 3100, "new": 1, "page": 16,
         "drop": 0.0},
        # a server's step that ends some requests and admits the prompts of others
        {"name": "plan_prompts", "op": "plan", "requests": 256, "held": 4096, "new": 2048,
         "page": 64, "drop": 0.5},
        # the same decode step's q/k norms, rotation and append
        {"name": "rotate_decode", "op": "rotate", "tokens": 8, "hq": 32, "hk": 8, "d": 128,
         "axes": 3, "page": 16, "norm": True},
        # a prompt of text and an image, as in a prefill
        {"name": "rotate_prompt", "op": "rotate", "tokens": 3100, "hq": 32, "hk": 8, "d": 128,
         "axes": 3, "page": 64, "norm": True},
        # the prompts of several requests at once
        {"name": "rotate_prompts", "op": "rotate", "tokens": 16381, "hq": 32, "hk": 8, "d": 128,
         "axes": 3, "page": 16, "norm": False},
        # a vision encoder's rows and columns, q and k of a packed projection, no cache
        {"name": "rotate_vision", "op": "rotate", "tokens": 16384, "hq": 16, "hk": 16, "d": 80,
         "axes": 2, "page": 0, "norm": False},
        # one decode step over the in-place cache of a prompt
        {"name": "attend_decode", "op": "attend", "batch": 1, "new": 1, "held": 3100, "ragged": False,
         "hq": 32, "hk": 8, "d": 128, "page": 0, "causal": True},
        # small heads, short requests, some of them just begun
        {"name": "attend_short", "op": "attend", "batch": 16, "new": 1, "held": 515, "ragged": True,
         "hq": 8, "hk": 2, "d": 64, "page": 16, "causal": True},
        # one decode step of a server's 64 requests of all lengths
        {"name": "attend_batch", "op": "attend", "batch": 64, "new": 1, "held": 8192, "ragged": True,
         "hq": 32, "hk": 8, "d": 128, "page": 16, "causal": True},
        # two requests with very long contexts
        {"name": "attend_long", "op": "attend", "batch": 2, "new": 1, "held": 131001, "ragged": False,
         "hq": 32, "hk": 8, "d": 128, "page": 64, "causal": True},
        # an action expert's step: its tokens see the prompt and each other
        {"name": "attend_flow", "op": "attend", "batch": 1, "new": 32, "held": 3126, "ragged": False,
         "hq": 32, "hk": 8, "d": 128, "page": 0, "causal": False},
        # chunks of four prompts over what they hold already
        {"name": "attend_chunk", "op": "attend", "batch": 4, "new": 128, "held": 6100, "ragged": True,
         "hq": 32, "hk": 8, "d": 128, "page": 64, "causal": True},
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(("plan", "rotate", "rotate", "attend", "attend", "attend"))
    if op == "plan":
        return {"op": op, "requests": _log(rng, 1, 256), "held": _log(rng, 1, 4096),
                "new": rng.choice((1, _log(rng, 1, 2048))), "page": rng.choice((16, 32, 64, 128)),
                "drop": rng.choice((0.0, 0.25, 0.5))}
    if op == "rotate":
        if rng.random() < 0.3:
            heads, d = rng.choice(((16, 80), (16, 64), (12, 128)))
            return {"op": op, "tokens": _log(rng, 64, 16384), "hq": heads, "hk": heads, "d": d,
                    "axes": 2, "page": 0, "norm": False}
        hq, hk, d = rng.choice(((32, 8, 128), (16, 8, 128), (8, 2, 64), (14, 2, 64), (8, 4, 256)))
        return {"op": op, "tokens": _log(rng, 1, 16384), "hq": hq, "hk": hk, "d": d, "axes": 3,
                "page": rng.choice((16, 32, 64, 128)), "norm": rng.random() < 0.5}
    hq, hk, d = rng.choice(((32, 8, 128), (32, 8, 128), (16, 8, 128), (8, 8, 128), (8, 2, 64),
                            (14, 2, 64), (8, 4, 256), (16, 1, 256)))
    new = rng.choice((1, 1, _log(rng, 2, 128)))
    # what is read stays below the long requests', what is multiplied below the chunks'
    held = _log(rng, 1, 131072 if new == 1 else 6100)
    most = 262000 * 8 * 128 // (held * hk * d) if new == 1 else 4 * 128 * 6100 * 32 * 128 // (new * held * hq * d)
    return {"op": op, "batch": _log(rng, 1, max(1, min(64, most))), "new": new, "held": max(held, new),
            "ragged": rng.random() < 0.7, "hq": hq, "hk": hk, "d": d,
            "page": rng.choice((0, 16, 32, 64, 128)), "causal": rng.random() < 0.8}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _gpu(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, *shape, scale=1.0, shift=0.0):
    return torch.randn(*shape, generator=g, device=DEV).mul_(scale).add_(shift).to(BF)


def _spread(n, hi, salt=0):
    """n lengths of at most hi, their logarithms spread evenly; one is hi.  The same ones for
    every seed, which decides their order."""
    rng = random.Random(n * 1000003 + hi * 101 + salt)
    return [hi] + [max(1, round(hi ** rng.random())) for _ in range(n - 1)]


def _requests(case):
    """(tokens held, tokens kept, new tokens) of each request of a plan.  A request that ends
    gives its place to a prompt; one that goes on has one new token, or a prompt's next chunk."""
    n, rng = case["requests"], random.Random(case["requests"] + case["held"])
    held = _spread(n, case["held"])
    drop = [rng.random() < case["drop"] for _ in range(n)]
    new = [1] * n if case["new"] == 1 else _spread(n, case["new"], 1)
    if case["drop"]:
        new = [x if d else 1 for x, d in zip(new, drop)]
    return [(h, 0 if d else h, x) for h, d, x in zip(held, drop, new)]


def _pages(seed, counts, more):
    """A table whose requests hold counts[r] pages of a shuffled pool with `more` free ones:
    (table [R, W], ring [P], free pages)."""
    rng = np.random.RandomState(int(seed) & 0x7FFFFFFF)
    total = sum(counts) + more
    order = rng.permutation(total).astype(np.int32)
    table = np.zeros((len(counts), max(counts)), np.int32)
    at = 0
    for r, c in enumerate(counts):
        table[r, :c] = order[at:at + c]
        at += c
    ring = np.full(total, -1, np.int32)
    ring[:more] = order[at:]
    return table, ring, more


def _grid_positions(tokens, axes, seed):
    """Positions [axes, tokens] of a prompt: text, an image of rows and columns, text (three
    axes); or the patches of an image (two)."""
    n = np.arange(tokens, dtype=np.int64)
    if axes == 2:
        side = max(1, round(tokens ** 0.5))
        return np.stack((n // side, n % side))
    if tokens < 64:  # tokens of a decode step, each of a request of its own
        return np.broadcast_to(np.random.RandomState(int(seed) & 0x7FFFFFFF).randint(0, 40000, tokens),
                               (3, tokens)).astype(np.int64)
    lead, cols = tokens // 8, max(1, round((tokens // 2) ** 0.5))
    rows = (tokens // 2) // cols
    image = rows * cols
    j = np.arange(image)
    mid = np.stack((np.full(image, lead), lead + j // cols, lead + j % cols))
    tail = lead + max(rows, cols) + np.arange(tokens - lead - image)
    return np.concatenate((np.broadcast_to(n[:lead], (3, lead)), mid,
                           np.broadcast_to(tail, (3, len(tail)))), axis=1).astype(np.int64)


def _frequencies(case):
    """(inv_freq [D/2] fp32, axis [D/2]): which axis turns which pair, and how fast."""
    d, half = case["d"], case["d"] // 2
    if case["axes"] == 2:  # the first half of the pairs by rows, the second by columns
        quarter = half // 2
        inv = THETA["vision"] ** (-np.arange(quarter) * 2.0 / half)
        return np.concatenate((inv, inv)).astype(np.float32), np.repeat((0, 1), quarter)
    inv = THETA["text"] ** (-np.arange(half) * 2.0 / d)
    axis = np.zeros(half, np.int64)  # height and width take every third pair, time the rest
    for a in (1, 2):
        axis[a:3 * SECTIONS[d][a]:3] = a
    return inv.astype(np.float32), axis


def _inputs(case, seed):
    rng, g = random.Random(int(seed)), _gpu(seed)
    op = case["op"]
    if op == "plan":
        n, ps, each = case["requests"], case["page"], _requests(case)
        rng.shuffle(each)
        have = [-(-h // ps) for h, _, _ in each]
        need = [-(-(k + x) // ps) for _, k, x in each]
        table, ring, free = _pages(seed, have, sum(need) + 8)
        wide = np.zeros((n, max(max(have), max(need))), np.int32)
        wide[:, :table.shape[1]] = table
        ints = {"held": [h for h, _, _ in each], "new": [x for _, _, x in each],
                # one that goes on keeps whatever it holds
                "keep": [k if k == 0 else 1 << 30 for _, k, _ in each],
                "delta": [rng.randint(-500, 0) for _ in range(n)]}
        # room for some more tokens than come
        return {"host": ints, "free": free, "table": wide, "ring": ring,
                "tokens": sum(ints["new"]) + (n if case["drop"] else 0)}
    if op == "rotate":
        t, hq, hk, d, ps = case["tokens"], case["hq"], case["hk"], case["d"], case["page"]
        pos = _grid_positions(t, case["axes"], seed)
        inv, axis = _frequencies(case)
        s = {"pos": pos, "inv": inv, "axis": axis}
        if not ps:  # the encoder's packed projection
            qkv = _randn(g, t, 3, hq, d)
            return {**s, "q": qkv[:, 0], "k": qkv[:, 1]}
        pages = -(-t // ps) + 4
        slot = np.random.RandomState(int(seed) & 0x7FFFFFFF).permutation(pages)[:-(-t // ps), None] * ps
        slot = (slot + np.arange(ps)).reshape(-1)[:t].astype(np.int64)
        s |= {"q": _randn(g, t, hq, d), "k": _randn(g, t, hk, d), "v": _randn(g, t, hk, d),
              "slot": slot, "pages": pages}
        if case["norm"]:
            s |= {"qw": _randn(g, d, scale=0.1, shift=1.0), "kw": _randn(g, d, scale=0.1, shift=1.0)}
        return s
    b, s, hq, hk, d, ps = (case[k] for k in ("batch", "new", "hq", "hk", "d", "page"))
    # a request that has fewer new tokens than the others leaves rows empty
    held = _spread(b, case["held"]) if case["ragged"] else [case["held"]] * b
    rng.shuffle(held)
    some = [min(s, h) for h in held]
    q = _randn(g, b, s, hq, d, scale=1.5).transpose(1, 2)
    if ps:
        counts = [-(-h // ps) for h in held]
        table, _, _ = _pages(seed, counts, 3)
        shape = (sum(counts) + 3, hk, ps, d)
    else:
        table, shape = None, (b, hk, max(held) + 8, d)
    return {"q": q, "k": _randn(g, *shape), "v": _randn(g, *shape), "table": table, "held": held,
            "some": some}


def _dev(a, dtype=None):
    return torch.as_tensor(np.ascontiguousarray(a), dtype=dtype, device=DEV)


def prepare(case, seed):
    x = _inputs(case, seed)
    op, i32 = case["op"], torch.int32
    s = {"case": case}
    if op == "plan":
        s |= {k: _dev(v, i32) for k, v in x["host"].items()}
        s |= {"table": _dev(x["table"]), "ring": _dev(x["ring"]), "tokens": x["tokens"],
              "cursor": _dev([0, x["free"], 0, 0], i32)}
        return s
    if op == "rotate":
        s |= {k: x[k] for k in ("q", "k", "v", "qw", "kw") if k in x}
        s |= {"pos": _dev(x["pos"]), "inv": _dev(x["inv"]), "axis": _dev(x["axis"])}
        if case["page"]:
            shape = (x["pages"], case["hk"], case["page"], case["d"])
            s |= {"slot": _dev(x["slot"]), "kp": torch.zeros(shape, dtype=BF, device=DEV),
                  "vp": torch.zeros(shape, dtype=BF, device=DEV)}
        if own:  # which pair turns with which axis, laid out once for all calls
            s["plan"] = _package().axial.AxisPlan(s["inv"], s["axis"])
        return s
    s |= {k: x[k] for k in ("q", "k", "v", "held", "some")}
    s |= {"lens": _dev(x["held"], i32), "news": _dev(x["some"], i32),
          "table": None if x["table"] is None else _dev(x["table"])}
    return s


@functools.lru_cache(maxsize=None)
def _package():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    at = os.path.join(root, "umic-alpamayo_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from umic import kernels
    from umic.kernels import attention, axial, paged  # noqa: F401

    return kernels


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

@torch.no_grad()
def run(state):
    case = state["case"]
    return (_OWN if own else _PLAIN)[case["op"]](case, state)


def _own_plan(case, s):
    step = _package().paged.plan_pages(s["held"], s["new"], s["table"], s["ring"], s["cursor"],
                                       case["page"], s["tokens"], keep=s["keep"], delta=s["delta"])
    return [step.kv_len, step.cursor, step.starts, step.slots, step.positions, s["table"], s["ring"]]


def _own_rotate(case, s):
    axial = _package().axial
    norm = (s["qw"], s["kw"], EPS) if case["norm"] else None
    if not case["page"]:
        return axial.rotate(s["q"], s["k"], s["pos"], s["plan"], norm)
    q = axial.rotate_append(s["q"], s["k"], s["v"], s["pos"], s["plan"], s["slot"], s["kp"], s["vp"],
                            norm)
    return q, s["kp"], s["vp"]


def _own_attend(case, s):
    # lengths that are the same for all are known to the host
    lens = s["lens"] if case["ragged"] else case["held"]
    news = s["news"] if case["ragged"] and case["new"] > 1 else None
    return _package().attention.cache_attention(s["q"], s["k"], s["v"], lens, table=s["table"],
                                                q_len=news, causal=case["causal"])


def _plain_plan(case, s):
    ps, table, ring = case["page"], s["table"], s["ring"]
    held, new, total = s["held"].long(), s["new"].long(), ring.numel()
    head, free = s["cursor"][0].long(), s["cursor"][1].long()
    kept = torch.minimum(s["keep"].long().clamp(min=0), held)
    have, length = (held + ps - 1) // ps, kept + new
    need = (length + ps - 1) // ps
    w = torch.arange(table.shape[1], device=table.device)[None]
    back, take = (w >= need[:, None]) & (w < have[:, None]), (w >= have[:, None]) & (w < need[:, None])
    order = back.flatten().cumsum(0) - 1
    at = (head + free + order)[back.flatten()] % total
    ring[at] = table[back]
    order = take.flatten().cumsum(0) - 1
    table[take] = ring[(head + order)[take.flatten()] % total]
    starts = torch.cat((new.new_zeros(1), new.cumsum(0)))
    t = torch.arange(s["tokens"], device=table.device)
    r = (torch.searchsorted(starts, t, right=True) - 1).clamp(max=held.numel() - 1)
    pos = (kept[r] + t - starts[r]).clamp(max=table.shape[1] * ps - 1)
    real = t < starts[-1]
    slots = torch.where(real, table[r, pos // ps].long() * ps + pos % ps, -1)
    pos = torch.where(real, pos + s["delta"].long()[r], 0)
    took, gave = take.sum(), back.sum()
    cursor = torch.stack(((head + took) % total, free + gave - took, starts[-1], starts[-1] * 0))
    i32 = torch.int32
    return [length.to(i32), cursor.to(i32), starts.to(i32), slots, pos, table, ring]


def _plain_norm(x, w):
    x = x.float()
    return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()


def _turn(x, cos, sin):
    a, b = x.chunk(2, dim=-1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)


def _plain_rotate(case, s):
    angle = s["pos"][s["axis"]].t().double() * s["inv"].double()  # far positions lose bits in 32
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    q = _turn(_plain_norm(s["q"], s.get("qw")), cos, sin).to(BF)
    k = _turn(_plain_norm(s["k"], s.get("kw")), cos, sin).to(BF)
    if not case["page"]:
        return q, k
    page, row = s["slot"] // case["page"], s["slot"] % case["page"]
    s["kp"][page, :, row] = k
    s["vp"][page, :, row] = s["v"]
    return q, s["kp"], s["vp"]


def _rows(cache, table, b, n):
    """The n rows [Hk, n, D] that request b holds."""
    if table is None:
        return cache[b, :, :n]
    pages = cache[table[b, :-(-n // cache.shape[2])].long()]
    return pages.transpose(0, 1).reshape(cache.shape[1], -1, cache.shape[3])[:, :n]


def _visible(case, some, n, dev):
    """[some, n]: which of a request's keys its new tokens see."""
    i, j = torch.arange(some, device=dev)[:, None], torch.arange(n, device=dev)[None]
    return j <= n - some + i if case["causal"] else (j < n).expand(some, n)


def _softmax_product(case, q, k, v, some):
    """q [Hq, some, D] over k, v [Hk, n, D] of the same type."""
    hk, n, d = k.shape
    q = q.reshape(hk, -1, d)
    x = torch.matmul(q, k.transpose(1, 2).contiguous()) * (1.0 / math.sqrt(d))
    if case["causal"] and some > 1:
        see = _visible(case, some, n, x.device).repeat(q.shape[1] // some, 1)
        x = x.masked_fill(~see, -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    return (torch.matmul(p, v) / p.sum(-1, keepdim=True)).reshape(-1, some, d)


def _attend(case, s, kind):
    b, n, hq, d = case["batch"], case["new"], case["hq"], case["d"]
    out = torch.zeros(b, n, hq, d, dtype=BF if kind is torch.float32 else kind, device=DEV)
    for i, (held, some) in enumerate(zip(s["held"], s["some"])):
        k, v = (_rows(s[x], s["table"], i, held).to(kind) for x in ("k", "v"))
        o = _softmax_product(case, s["q"][i, :, :some].to(kind), k, v, some)
        out[i, :some] = o.transpose(0, 1)
    return out


def _plain_attend(case, s):
    return _attend(case, s, torch.float32)


_PLAIN = {"plan": _plain_plan, "rotate": _plain_rotate, "attend": _plain_attend}
_OWN = {"plan": _own_plan, "rotate": _own_rotate, "attend": _own_attend}


# ---------------------------------------------------------------------------
# What a pass cannot do without, and its values in 64 bits
# ---------------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "plan":
        n, ps, each = case["requests"], case["page"], _requests(case)
        tokens = sum(x for _, _, x in each)
        moved = sum(abs(-(-(k + x) // ps) - -(-h // ps)) for h, k, x in each)
        # lengths in and out, slots and positions out, the pages that move
        return {"bytes": 4 * 7 * n + 16 * tokens + 8 * moved, "flops": 8 * tokens}
    if op == "rotate":
        t, hq, hk, d = (case[k] for k in ("tokens", "hq", "hk", "d"))
        moved = hq + (2 * hk if case["page"] else hk)
        return {"bytes": 4 * t * moved * d + 8 * t * (case["axes"] + (1 if case["page"] else 0)),
                "flops": t * (hq + hk) * d * (7 if case["norm"] else 3)}
    b, s, hq, hk, d = (case[k] for k in ("batch", "new", "hq", "hk", "d"))
    rows = sum(_spread(b, case["held"])) if case["ragged"] else b * case["held"]
    return {"bytes": int(4 * rows * hk * d + 4 * b * s * hq * d), "flops": int(4 * rows * s * hq * d)}


def _exact_plan(case, x):
    """Request by request, on the host."""
    ps, h = case["page"], x["host"]
    table, ring = x["table"].copy(), x["ring"].copy()
    total, tail, head = len(ring), x["free"], 0
    spans = [(min(max(k, 0), n), n, min(max(k, 0), n) + m)
             for k, n, m in zip(h["keep"], h["held"], h["new"])]
    for r, (_, n, after) in enumerate(spans):
        for w in range(-(-after // ps), -(-n // ps)):
            ring[tail % total] = table[r, w]
            tail += 1
    slots, pos, starts = [], [], [0]
    for r, (kept, n, after) in enumerate(spans):
        for w in range(-(-n // ps), -(-after // ps)):
            table[r, w] = ring[head % total]
            head += 1
        p = np.arange(kept, after)
        slots.append(table[r, p // ps].astype(np.int64) * ps + p % ps)
        pos.append(p + h["delta"][r])
        starts.append(starts[-1] + len(p))
    cursor = [head % total, tail - head, starts[-1], 0]
    spare = x["tokens"] - starts[-1]
    slots.append(np.full(spare, -1))
    pos.append(np.zeros(spare, np.int64))
    return [np.array([a for _, _, a in spans], np.int32), np.array(cursor, np.int32),
            np.array(starts, np.int32), np.concatenate(slots), np.concatenate(pos).astype(np.int64),
            table, ring]


@torch.no_grad()
def exact(case, seed):
    x = _inputs(case, seed)
    if case["op"] == "plan":
        return _exact_plan(case, x)
    if case["op"] == "rotate":
        pos, inv, axis = _dev(x["pos"]).double(), _dev(x["inv"]).double(), _dev(x["axis"])
        turn = torch.polar(torch.ones_like(inv), inv * 0)[None] * torch.exp(1j * pos[axis].t() * inv)

        def rotated(y, w):
            y = y.double()
            if w is not None:
                y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * w.double()
            half = y.shape[-1] // 2
            z = torch.complex(y[..., :half].contiguous(), y[..., half:].contiguous()) * turn[:, None]
            return torch.cat((z.real, z.imag), dim=-1)

        q, k = rotated(x["q"], x.get("qw")), rotated(x["k"], x.get("kw"))
        if not case["page"]:
            return q, k
        shape = (x["pages"] * case["page"], case["hk"], case["d"])
        pools = []
        for rows in (k, x["v"].double()):
            flat = torch.zeros(shape, dtype=torch.float64, device=DEV)
            flat[_dev(x["slot"])] = rows
            pools.append(flat.view(x["pages"], case["page"], *shape[1:]).transpose(1, 2))
        return q, *pools
    table = None if x["table"] is None else _dev(x["table"])
    out = torch.zeros(case["batch"], case["new"], case["hq"], case["d"], dtype=torch.float64, device=DEV)
    group = case["hq"] // case["hk"]
    for i, (held, some) in enumerate(zip(x["held"], x["some"])):
        k, v = (_rows(x[y], table, i, held) for y in ("k", "v"))
        see = _visible(case, some, held, DEV)
        for h in range(case["hk"]):
            q = x["q"][i, h * group:(h + 1) * group, :some].double()
            logit = (q @ k[h].double().t()) * case["d"] ** -0.5
            logit = torch.where(see, logit, torch.full_like(logit, -math.inf))
            out[i, :some, h * group:(h + 1) * group] = (torch.softmax(logit, -1) @ v[h].double()).transpose(0, 1)
    return out
