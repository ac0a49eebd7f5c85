"""The 8-bit paged cache's operators as timed cases: new tokens rotated and written as
codes with a scale for each block of 16 tokens and key head, rows read back as bf16, and
attention of new tokens over the codes.

A block's scale is a power of two, so that a code times its scale is a bf16 number.  `own`
false computes all of it in elementary torch operations, in 32 bits (angles in 64); `own`
true makes the package's calls.  The sizes are the package's own (a text trunk of 32 query
and 8 key / value heads of 128, a prompt of about 3100 tokens, an action expert of 32
tokens a step) and generic ones for a server of many requests.
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
THETA = 1e6
SECTIONS = {128: (24, 20, 20), 64: (12, 10, 10), 256: (48, 40, 40)}  # time, height, width
BLOCK = 16        # tokens that share a scale
LEAST = -100      # exponent of the smallest scale
TYPES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
BITS = {"int8": 6, "e4m3": 7}  # a block's largest value is 2^BITS to 2^(BITS + 1) codes


def listed():
    return [
        # one decode step of eight requests: a token each, into blocks that hold some already
        {"name": "write_decode", "op": "write", "kind": "int8", "batch": 8, "tokens": 8,
         "held": 3100, "hq": 32, "hk": 8, "d": 128, "page": 64, "turn": True, "norm": True},
        # a prompt of text and an image, as in a prefill
        {"name": "write_prompt", "op": "write", "kind": "int8", "batch": 1, "tokens": 3100,
         "held": 0, "hq": 32, "hk": 8, "d": 128, "page": 64, "turn": True, "norm": True},
        # the next chunks of several prompts at once
        {"name": "write_prompts", "op": "write", "kind": "e4m3", "batch": 5, "tokens": 16381,
         "held": 515, "hq": 32, "hk": 8, "d": 128, "page": 16, "turn": True, "norm": False},
        # keys that another model part has rotated, of small heads
        {"name": "write_plain", "op": "write", "kind": "e4m3", "batch": 3, "tokens": 1537,
         "held": 77, "hq": 14, "hk": 2, "d": 64, "page": 32, "turn": False, "norm": False},
        # sixteen short requests back as bf16, for a computation that has no 8-bit form
        {"name": "read_short", "op": "read", "kind": "e4m3", "batch": 16, "held": 515,
         "ragged": True, "hk": 2, "d": 64, "page": 16},
        # a few long ones, as they are handed on to another cache
        {"name": "read_long", "op": "read", "kind": "int8", "batch": 4, "held": 30011,
         "ragged": False, "hk": 8, "d": 128, "page": 64},
        # one decode step over a prompt
        {"name": "attend_decode", "op": "attend", "kind": "int8", "batch": 1, "new": 1,
         "held": 3100, "ragged": False, "hq": 32, "hk": 8, "d": 128, "page": 64, "causal": True},
        # one decode step of a server's 64 requests of all lengths
        {"name": "attend_batch", "op": "attend", "kind": "e4m3", "batch": 64, "new": 1,
         "held": 8192, "ragged": True, "hq": 32, "hk": 8, "d": 128, "page": 16, "causal": True},
        # two requests with very long contexts, in either type
        {"name": "attend_long", "op": "attend", "kind": "int8", "batch": 2, "new": 1,
         "held": 131001, "ragged": False, "hq": 32, "hk": 8, "d": 128, "page": 64, "causal": True},
        {"name": "attend_long_e4m3", "op": "attend", "kind": "e4m3", "batch": 2, "new": 1,
         "held": 131001, "ragged": False, "hq": 32, "hk": 8, "d": 128, "page": 64, "causal": True},
        # an action expert's step: its tokens see the prompt and each other
        {"name": "attend_flow", "op": "attend", "kind": "int8", "batch": 1, "new": 32,
         "held": 3126, "ragged": False, "hq": 32, "hk": 8, "d": 128, "page": 64, "causal": False},
        # chunks of four prompts over what they hold already
        {"name": "attend_chunk", "op": "attend", "kind": "e4m3", "batch": 4, "new": 128,
         "held": 6100, "ragged": True, "hq": 32, "hk": 8, "d": 128, "page": 64, "causal": True},
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(("write", "write", "read", "attend", "attend", "attend"))
    kind = rng.choice(("int8", "e4m3"))
    page = rng.choice((16, 32, 64, 128))
    if op == "write":
        hq, hk, d = rng.choice(((32, 8, 128), (16, 8, 128), (8, 2, 64), (14, 2, 64), (8, 4, 256)))
        tokens = _log(rng, 1, 16381)
        turn = rng.random() < 0.7
        return {"op": op, "kind": kind, "batch": min(tokens, _log(rng, 1, 64)), "tokens": tokens,
                "held": rng.choice((0, _log(rng, 1, 4096))), "hq": hq, "hk": hk, "d": d,
                "page": page, "turn": turn, "norm": turn and rng.random() < 0.5}
    if op == "read":
        hk, d = rng.choice(((8, 128), (8, 128), (2, 64), (4, 256), (1, 256)))
        held = _log(rng, 1, 120000)
        return {"op": op, "kind": kind, "batch": _log(rng, 1, max(1, min(64, 120000 // held))),
                "held": held, "ragged": rng.random() < 0.5, "hk": hk, "d": d, "page": page}
    hq, hk, d = rng.choice(((32, 8, 128), (32, 8, 128), (16, 8, 128), (8, 8, 128), (8, 2, 64),
                            (14, 2, 64), (8, 4, 256), (16, 1, 256)))
    new = rng.choice((1, 1, _log(rng, 2, 128)))
    # what is read stays below the long requests', what is multiplied below the chunks'
    held = _log(rng, 1, 131072 if new == 1 else 6100)
    most = 262000 * 8 * 128 // (held * hk * d) if new == 1 else 4 * 128 * 6100 * 32 * 128 // (new * held * hq * d)
    return {"op": op, "kind": kind, "batch": _log(rng, 1, max(1, min(64, most))), "new": new,
            "held": max(held, new), "ragged": rng.random() < 0.7, "hq": hq, "hk": hk, "d": d,
            "page": page, "causal": rng.random() < 0.8}


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


def _shares(n, total):
    """n parts of total, one at least each, of different sizes."""
    rng = random.Random(n * 7919 + total)
    cuts = sorted(rng.sample(range(1, total), n - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def _requests(case):
    """(tokens held, new tokens) of each request."""
    n = case["batch"]
    if case["op"] == "write":
        held = _spread(n, case["held"]) if case["held"] else [0] * n
        return list(zip(held, _shares(n, case["tokens"])))
    held = _spread(n, case["held"]) if case.get("ragged") else [case["held"]] * n
    return [(h, 0) for h in held]


def _pages(seed, counts, more):
    """A table whose requests hold counts[r] pages of a shuffled pool with `more` others."""
    order = np.random.RandomState(int(seed) & 0x7FFFFFFF).permutation(sum(counts) + more)
    table = np.zeros((len(counts), max(max(counts), 1)), np.int32)
    at = 0
    for r, c in enumerate(counts):
        table[r, :c] = order[at:at + c]
        at += c
    return table


def _grid_positions(tokens, seed):
    """Positions [3, tokens] of a prompt: text, an image of rows and columns, text."""
    n = np.arange(tokens, dtype=np.int64)
    if tokens < 64:  # tokens of a decode step, each of a request of its own
        one = np.random.RandomState(int(seed) & 0x7FFFFFFF).randint(0, 40000, tokens)
        return np.broadcast_to(one, (3, tokens)).astype(np.int64)
    lead, cols = tokens // 8, max(1, round((tokens // 2) ** 0.5))
    rows = (tokens // 2) // cols
    j = np.arange(rows * cols)
    image = np.stack((np.full(len(j), lead), lead + j // cols, lead + j % cols))
    tail = lead + max(rows, cols) + np.arange(tokens - lead - len(j))
    return np.concatenate((np.broadcast_to(n[:lead], (3, lead)), image,
                           np.broadcast_to(tail, (3, len(tail)))), axis=1).astype(np.int64)


def _frequencies(d):
    """(inv_freq [D/2] fp32, axis [D/2]): height and width turn every third pair, time the rest."""
    half = d // 2
    inv = THETA ** (-np.arange(half) * 2.0 / d)
    axis = np.zeros(half, np.int64)
    for a in (1, 2):
        axis[a:3 * SECTIONS[d][a]:3] = a
    return inv.astype(np.float32), axis


def _exponents(kind, most):
    """Exponents of the scales of blocks whose largest magnitude is `most`."""
    return (torch.frexp(most.float())[1] - 1 - BITS[kind]).masked_fill(most == 0, LEAST).clamp(min=LEAST)


def _power(e):
    return torch.ldexp(torch.ones(e.shape, device=e.device), e)


def _codes(kind, x):
    """Codes of x, in units of its scale."""
    return (x.round().clamp(-127, 127) if kind == "int8" else x).to(TYPES[kind])


def _held_cache(case, g, pages):
    """Codes and scales of a pool of `pages` pages: tokens of different sizes, some columns
    larger than the others."""
    kind, shape = case["kind"], (pages, case["hk"], case["page"] // BLOCK, BLOCK, case["d"])
    codes, scales = [], []
    for _ in range(2):
        x = torch.randn(shape, generator=g, device=DEV)
        x *= torch.exp(0.5 * torch.randn(1, shape[1], 1, 1, shape[4], generator=g, device=DEV))
        scale = _power(_exponents(kind, x.abs().amax((3, 4))))
        codes.append(_codes(kind, x / scale[..., None, None]).view(pages, shape[1], case["page"], -1))
        scales.append(scale)
    return codes, scales


def _inputs(case, seed):
    rng, g = random.Random(int(seed)), _gpu(seed)
    op, ps, d, hk = case["op"], case["page"], case["d"], case["hk"]
    each = _requests(case)
    rng.shuffle(each)
    counts = [-(-(h + x) // ps) for h, x in each]
    table = _pages(seed, counts, 3)
    (k8, v8), (ks, vs) = _held_cache(case, g, sum(counts) + 3)
    s = {"k8": k8, "v8": v8, "ks": ks, "vs": vs, "table": table,
         "held": np.array([h for h, _ in each]), "kv": np.array([h + x for h, x in each])}
    if op == "write":
        t = case["tokens"]
        p = np.concatenate([np.arange(h, h + x) for h, x in each])
        r = np.repeat(np.arange(len(each)), [x for _, x in each])
        s |= {"slot": table[r, p // ps].astype(np.int64) * ps + p % ps,
              "k": _randn(g, t, hk, d), "v": _randn(g, t, hk, d)}
        # from the first block that is written on: what the write may change
        s |= {"start": s["held"] // BLOCK * BLOCK}
        s["rows"] = int((s["kv"] - s["start"]).max())
        if case["turn"]:
            s["q"] = _randn(g, t, case["hq"], d)
            s["pos"] = _grid_positions(t, seed)
            s["inv"], s["axis"] = _frequencies(d)
        if case["norm"]:
            s |= {"qw": _randn(g, d, scale=0.1, shift=1.0), "kw": _randn(g, d, scale=0.1, shift=1.0)}
    elif op == "read":
        s["rows"] = case["held"]
    else:
        b, n = case["batch"], case["new"]
        # a request that has fewer new tokens than the others leaves rows empty
        s["some"] = np.minimum(n, s["held"])
        s["q"] = _randn(g, b, n, case["hq"], d, scale=1.5).transpose(1, 2)
    return s


def _dev(a, dtype=None):
    return torch.as_tensor(np.ascontiguousarray(a), dtype=dtype, device=DEV)


def prepare(case, seed):
    s = _inputs(case, seed)
    i32 = torch.int32
    for key in ("table", "kv", "start", "some"):
        if key in s:
            s[key] = _dev(s[key], i32)
    for key in ("slot", "pos", "inv", "axis"):
        if key in s:
            s[key] = _dev(s[key])
    s["case"] = case
    if own:  # which pair turns with which axis, laid out once for all calls
        s["cache"] = _package().cache8.Pages8(s["k8"], s["v8"], s["ks"], s["vs"])
        if "pos" in s:
            s["plan"] = _package().axial.AxisPlan(s["inv"], s["axis"])
    return s


@functools.lru_cache(maxsize=None)
def _package():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    at = os.path.join(root, "umic-alpamayo_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from umic import kernels
    from umic.kernels import axial, cache8  # noqa: F401

    return kernels


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

@torch.no_grad()
def run(state):
    case = state["case"]
    return (_OWN if own else _PLAIN)[case["op"]](case, state)


def _own_write(case, s):
    """The new tokens' rows, and the rows of the blocks that they came into."""
    cache8, q = _package().cache8, ()
    if case["turn"]:
        norm = (s["qw"], s["kw"], EPS) if case["norm"] else None
        q = (cache8.rotate_append(s["q"], s["k"], s["v"], s["pos"], s["plan"], s["slot"], s["cache"],
                                  norm),)
    else:
        cache8.append(s["k"], s["v"], s["slot"], s["cache"])
    return *q, *cache8.read(s["cache"], s["table"], s["kv"], s["rows"], start=s["start"])


def _own_read(case, s):
    return _package().cache8.read(s["cache"], s["table"], s["kv"], s["rows"])


def _own_attend(case, s):
    # lengths that are the same for all are known to the host
    lens = s["kv"] if case["ragged"] else case["held"]
    news = s["some"] if case["ragged"] and case["new"] > 1 else None
    return _package().cache8.attention(s["q"], s["cache"], lens, s["table"], q_len=news,
                                       causal=case["causal"])


def _plain_norm(x, w):
    x = x.float()
    return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()


def _turn(x, cos, sin):
    a, b = x.chunk(2, dim=-1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)


def _plain_store(case, s, x, codes, scales):
    """Rows x [T, Hk, D] into their slots."""
    kind, ps, slot = case["kind"], case["page"], s["slot"]
    pages, hk, _, d = codes.shape
    per = ps // BLOCK
    page, row = slot // ps, slot % ps
    x = x.float()
    # [page, block, head]: the largest value that comes, and the first row that is written
    most = torch.zeros(pages * per, hk, device=DEV)
    most.index_reduce_(0, slot // BLOCK, x.abs().amax(-1), "amax")
    least = torch.full((pages * per,), BLOCK, device=DEV)
    least.index_reduce_(0, slot // BLOCK, slot % BLOCK, "amin")
    most = most.view(pages, per, hk).transpose(1, 2)
    least = least.view(pages, 1, per)
    e = _exponents(kind, most)
    before = torch.frexp(scales)[1] - 1
    e = torch.where((least > 0) & (least < BLOCK), torch.maximum(e, before), e)
    e = torch.where(least < BLOCK, e, before)
    # the rows before: of each request's first block
    at, of = s["start"].long(), s["table"].long()
    at = at.clamp(max=of.shape[1] * ps - 1)
    page0, block0 = of.gather(1, at[:, None] // ps)[:, 0], at % ps // BLOCK
    rows = block0[:, None] * BLOCK + torch.arange(BLOCK, device=DEV)
    old = codes.view(torch.uint8)[page0[:, None], :, rows].view(codes.dtype).float()  # [B, 16, Hk, D]
    ratio = _power(before[page0, :, block0] - e[page0, :, block0])
    old = _codes(kind, old * ratio[:, None, :, None])
    keep = torch.arange(BLOCK, device=DEV)[None] < least[page0, 0, block0][:, None]
    keep &= least[page0, 0, block0][:, None] < BLOCK
    old = torch.where(keep[:, :, None, None], old.view(torch.uint8),
                      codes.view(torch.uint8)[page0[:, None], :, rows])
    codes.view(torch.uint8)[page0[:, None], :, rows] = old
    scales.copy_(_power(e))
    new = _codes(kind, x / scales[page, :, row // BLOCK][..., None])
    codes.view(torch.uint8)[page, :, row] = new.view(torch.uint8)


def _plain_write(case, s):
    k, q = s["k"], ()
    if case["turn"]:
        angle = s["pos"][s["axis"]].t().double() * s["inv"].double()  # far positions lose bits in 32
        cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
        q = (_turn(_plain_norm(s["q"], s.get("qw")), cos, sin).to(BF),)
        k = _turn(_plain_norm(k, s.get("kw")), cos, sin).to(BF)
    _plain_store(case, s, k, s["k8"], s["ks"])
    _plain_store(case, s, s["v"], s["v8"], s["vs"])
    return *q, *_plain_read(case, s)


def _plain_rows(case, s, codes, scales):
    """[B, Hk, W page, D] fp32: all that the table's pages hold."""
    of = s["table"].long()
    x = codes.view(torch.uint8)[of].view(codes.dtype).float()
    b, w, hk, ps, d = x.shape
    x = x.view(b, w, hk, ps // BLOCK, BLOCK, d) * scales[of][..., None, None]
    return x.transpose(1, 2).reshape(b, hk, w * ps, d)


def _plain_read(case, s):
    got = []
    for codes, scales in ((s["k8"], s["ks"]), (s["v8"], s["vs"])):
        x = _plain_rows(case, s, codes, scales)
        i = torch.arange(s["rows"], device=DEV)[None] + (s["start"][:, None] if "start" in s else 0)
        there = i < s["kv"][:, None]
        at = i.clamp(max=x.shape[2] - 1).expand(x.shape[0], -1)
        x = torch.gather(x, 2, at[:, None, :, None].expand(-1, x.shape[1], -1, x.shape[3]))
        got.append((x * there[:, None, :, None]).to(BF))
    return tuple(got)


def _plain_attend(case, s):
    k = _plain_rows(case, s, s["k8"], s["ks"])
    b, hk, n, d = k.shape
    q = s["q"].float().reshape(b, hk, -1, d)  # [B, Hk, G S, D]
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(d))
    x = x.view(b, case["hq"], case["new"], n)
    j = torch.arange(n, device=DEV)[None, None]
    i = torch.arange(case["new"], device=DEV)[None, :, None]
    kv, some = s["kv"][:, None, None], s["some"][:, None, None]
    see = (j < kv) & ((j <= kv - some + i) if case["causal"] else True)
    x = x.masked_fill(~see[:, None], -math.inf)
    x -= x.amax(-1, keepdim=True)
    p = x.exp_().view(b, hk, -1, n)
    del x, k
    v = _plain_rows(case, s, s["v8"], s["vs"])
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    o = o.view(b, case["hq"], case["new"], d).transpose(1, 2)
    return torch.where((i < some)[..., None], o, 0.0).to(BF)


_PLAIN = {"write": _plain_write, "read": _plain_read, "attend": _plain_attend}
_OWN = {"write": _own_write, "read": _own_read, "attend": _own_attend}


# ---------------------------------------------------------------------------
# What a pass cannot do without, and its values in 64 bits
# ---------------------------------------------------------------------------

def work(case):
    hk, d = case["hk"], case["d"]
    each = _requests(case)
    if case["op"] == "read":
        rows = sum(h for h, _ in each)  # codes and scales in; padded rows out
        return {"bytes": 2 * hk * (rows * d + rows // BLOCK * 4)
                + 4 * hk * d * case["batch"] * case["held"], "flops": 2 * rows * hk * d}
    if case["op"] == "write":
        t = case["tokens"]
        back = max(h + x - h // BLOCK * BLOCK for h, x in each)  # rows read back, of each request
        moved = (4 * case["hq"] * d + 24 if case["turn"] else 0) + 8 + 4 * hk * d + 2 * hk * d
        return {"bytes": t * moved + 2 * hk * (t + len(each) * BLOCK) * (d + 4 // BLOCK)
                + 4 * hk * d * len(each) * back,
                "flops": t * ((case["hq"] + hk) * d * (7 if case["norm"] else 3 if case["turn"] else 0)
                              + 4 * hk * d)}
    rows = sum(h for h, _ in each)
    b, s, hq = case["batch"], case["new"], case["hq"]
    return {"bytes": int(2 * hk * (rows * d + rows // BLOCK * 4) + 4 * b * s * hq * d),
            "flops": int(4 * rows * s * hq * d)}


def _exact_round(kind, x):
    """The value in 64 bits of the code nearest to x, in units of its scale."""
    if kind == "int8":
        return x.round().clamp(-127, 127)
    step = torch.ldexp(torch.ones_like(x), (torch.frexp(x)[1] - 4).clamp(min=-9))
    return (x / step).round() * step


def _exact_request(x, case, r, which):
    """The blocks [Hk, n, 16, D] that request r's pages hold, their exponents [Hk, n]."""
    ps = case["page"]
    pages = _dev(x["table"][r, :-(-int(x["kv"][r]) // ps)]).long()
    c = x[which + "8"].view(torch.uint8)[pages].view(TYPES[case["kind"]]).double()
    c = c.transpose(0, 1).reshape(case["hk"], -1, BLOCK, case["d"])
    scale = x[which + "s"][pages].double().transpose(0, 1).reshape(case["hk"], -1)
    return c * scale[..., None, None], torch.log2(scale)


def _exact_store(case, x, r, new, which):
    """Request r's rows [Hk, kv, D] after new [n, Hk, D] came behind what it held."""
    rows, e = _exact_request(x, case, r, which)
    held, kv = int(x["held"][r]), int(x["kv"][r])
    first, last = held // BLOCK, -(-kv // BLOCK)
    fill = torch.zeros(last * BLOCK - held, *new.shape[1:], dtype=torch.float64, device=DEV)
    fill[:kv - held] = new
    part = rows[:, first:last].clone(memory_format=torch.contiguous_format)
    flat = part.view(part.shape[0], -1, part.shape[3])
    flat[:, held - first * BLOCK:] = 0.0
    come = torch.zeros_like(part)
    come.view(flat.shape)[:, held - first * BLOCK:] = fill.transpose(0, 1)
    top = come.abs().amax((2, 3))
    up = torch.where(top > 0, torch.floor(torch.log2(top.clamp(min=1e-300))) - BITS[case["kind"]],
                     torch.full_like(top, LEAST)).clamp(min=LEAST)
    if held % BLOCK:
        up[:, 0] = torch.maximum(up[:, 0], e[:, first])
    step = torch.exp2(up)[..., None, None]
    return (_exact_round(case["kind"], (part + come) / step) * step).view(flat.shape)[:, :kv - first * BLOCK]


def _exact_write(case, x):
    q, k = [], x["k"].double()
    if case["turn"]:
        angle = _dev(x["pos"]).double()[_dev(x["axis"])].t() * _dev(x["inv"]).double()
        turn = torch.polar(torch.ones_like(angle), angle)[:, None]

        def rotated(y, w):
            y = y.double()
            if w is not None:
                y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * w.double()
            a, b = y[..., :case["d"] // 2], y[..., case["d"] // 2:]
            z = torch.complex(a.contiguous(), b.contiguous()) * turn
            return torch.cat((z.real, z.imag), dim=-1)

        q, k = [rotated(x["q"], x.get("qw"))], rotated(x["k"], x.get("kw")).to(BF).double()
    shape = (case["batch"], case["hk"], x["rows"], case["d"])
    got = [torch.zeros(shape, dtype=torch.float64, device=DEV) for _ in range(2)]
    at = 0
    for r in range(case["batch"]):
        n = int(x["kv"][r] - x["held"][r])
        for out, new, which in zip(got, (k, x["v"].double()), "kv"):
            rows = _exact_store(case, x, r, new[at:at + n], which)
            out[r, :, :rows.shape[1]] = rows
        at += n
    return *q, *got


@torch.no_grad()
def exact(case, seed):
    x = _inputs(case, seed)
    if case["op"] == "write":
        return _exact_write(case, x)
    if case["op"] == "read":
        shape = (case["batch"], case["hk"], x["rows"], case["d"])
        got = [torch.zeros(shape, dtype=torch.float64, device=DEV) for _ in range(2)]
        for r in range(case["batch"]):
            for out, which in zip(got, "kv"):
                n = int(x["kv"][r])
                out[r, :, :n] = _exact_request(x, case, r, which)[0].flatten(1, 2)[:, :n]
        return tuple(got)
    shape = (case["batch"], case["new"], case["hq"], case["d"])
    out = torch.zeros(shape, dtype=torch.float64, device=DEV)
    group = case["hq"] // case["hk"]
    for r in range(case["batch"]):
        n, some = int(x["kv"][r]), int(x["some"][r])
        k, v = (_exact_request(x, case, r, which)[0].flatten(1, 2)[:, :n] for which in "kv")
        i, j = torch.arange(some, device=DEV)[:, None], torch.arange(n, device=DEV)[None]
        hidden = (j > n - some + i) if case["causal"] else (j >= n).expand(some, n)
        for h in range(case["hk"]):
            q = x["q"][r, h * group:(h + 1) * group, :some].double()
            logit = (q @ k[h].t().contiguous()) / math.sqrt(case["d"])
            logit = logit.masked_fill(hidden, -math.inf)
            out[r, :some, h * group:(h + 1) * group] = (torch.softmax(logit, -1) @ v[h]).transpose(0, 1)
    return out
