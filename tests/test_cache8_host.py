"""What the 8-bit cache's operators refuse, before any launch (no GPU needed)."""

from __future__ import annotations

import copy
import ctypes

import pytest
import torch

from umic.kernels import axial, cache8
from umic.paged_cache import PagedArena, PagedKVCache

ARG, UNS = -1, -2
FAKE = 1 << 20  # aligned, never dereferenced: every call below returns early


@pytest.fixture(scope="module")
def lib():
    from umic import _lib

    return _lib.load()


def struct(**kw):
    """A cache's description, as (address, structure)."""
    from umic import _lib

    f = dict(k_codes=FAKE, v_codes=FAKE, k_scale=FAKE, v_scale=FAKE, pages=8, page_size=16, heads=2,
             head_dim=64, c_sb=2048, c_sh=1024, c_ss=64, s_sb=2, s_sh=1, format=1) | kw
    c = _lib.Cache8(**f)
    return ctypes.addressof(c), c


CACHE_ARG = [dict(pages=-1), dict(page_size=0), dict(heads=0), dict(head_dim=0), dict(k_codes=None),
             dict(v_codes=None), dict(k_scale=None), dict(v_scale=None)]
CACHE_UNS = [dict(head_dim=80), dict(head_dim=512), dict(page_size=8), dict(page_size=24),
             dict(page_size=1 << 31), dict(pages=1 << 31), dict(pages=1 << 30, page_size=32),
             dict(heads=1 << 17), dict(format=2), dict(format=-1), dict(c_sb=2056), dict(c_sh=1032),
             dict(c_ss=72), dict(k_codes=FAKE + 8), dict(v_codes=FAKE + 4)]


def test_cache_refusals(lib):
    """Each entry point's own look at a cache."""
    def each(**kw):
        at, keep = struct(**kw)
        return {lib.umic_cache8_append_bf16(at, *[FAKE] * 8, 1.0, None, None, 1e-6, 3, 4, 3, 3, 1,
                                            *[256, 64] * 3, None),
                lib.umic_cache8_read_bf16(at, *[FAKE] * 5, 2, 9, 4, 4, 9, None),
                lib.umic_cache8_attention_bf16(at, *[FAKE] * 5, 2, 1, 4, *[1024] * 6, 4, 4, 9, 1, 0.1,
                                               None, FAKE, 1 << 40, None)}

    for bad in CACHE_ARG:
        assert each(**bad) == {ARG}, bad
    for bad in CACHE_UNS:
        assert each(**bad) == {UNS}, bad


def test_append_refusals(lib):
    names = ("cache", "q", "k", "v", "qo", "pos", "turn", "axis", "slots")
    at, keep = struct()

    def f(T=3, Hq=4, axes=3, st=1024, qw=None, kw=None, **p):
        p = dict.fromkeys(names, FAKE) | {"cache": at} | p
        return lib.umic_cache8_append_bf16(*(p[n] for n in names), 1.0, qw, kw, 1e-6, T, Hq, axes, T,
                                           1, *[st, 64] * 3, None)

    assert f(T=-1) == f(Hq=-1) == f(axes=0) == ARG
    assert f(T=0, **dict.fromkeys(names[1:])) == 0
    for n in names:
        if n != "turn":
            assert f(**{n: None}) == ARG, n
    assert f(turn=None) == ARG                             # q without a rotation
    assert f(turn=None, Hq=0, kw=FAKE) == f(turn=None, Hq=0, qw=FAKE) == ARG
    assert f(qw=FAKE) == f(kw=FAKE) == ARG                 # one norm without the other
    assert f(st=1020) == f(k=FAKE + 8) == f(qo=FAKE + 2) == f(qw=FAKE + 8, kw=FAKE) == UNS
    assert f(Hq=1 << 17) == f(T=1 << 40) == UNS


def test_read_refusals(lib):
    at, keep = struct()
    none, none_keep = struct(pages=0)
    tall, tall_keep = struct(heads=1 << 15)

    def f(cache=at, B=2, rows=9, ld=4, w=4, n=9, lens=None, p=(FAKE,) * 3):
        return lib.umic_cache8_read_bf16(cache, *p, lens, None, B, rows, ld, w, n, None)

    assert f(B=-1) == f(rows=-1) == f(w=-1) == f(ld=3) == f(n=65) == f(n=-1) == f(none) == ARG
    assert f(B=0, p=(None,) * 3) == f(rows=0, p=(None,) * 3) == 0
    for i in range(3):
        assert f(p=tuple(None if j == i else FAKE for j in range(3))) == ARG, i
    assert f(w=1 << 40, ld=1 << 40) == f(B=1 << 21) == f(rows=1 << 32) == UNS
    assert f(tall, B=1 << 20) == UNS                       # more than a grid counts
    assert f(p=(FAKE + 8, FAKE, FAKE)) == f(p=(FAKE, FAKE + 8, FAKE)) == UNS


def test_attention_refusals(lib):
    at, keep = struct()
    odd, odd_keep = struct(heads=3)

    def f(cache=at, B=2, S=1, Hq=8, q=FAKE, out=FAKE, table=FAKE, lens=None, st=1024, ld=4, w=4, n=64,
          scale=0.1, ws=FAKE, size=1 << 40):
        return lib.umic_cache8_attention_bf16(cache, q, out, table, lens, None, B, S, Hq, st, st, 64,
                                              st, st, 64, ld, w, n, 1, scale, None, ws, size, None)

    assert f(B=-1) == f(S=-1) == f(Hq=-1) == f(size=-1) == f(None) == ARG
    assert f(B=0) == f(S=0) == f(Hq=0) == 0
    assert f(odd) == ARG
    assert f(q=None) == f(out=None) == f(ws=None) == f(table=None) == ARG
    assert f(scale=float("inf")) == f(scale=float("nan")) == ARG
    assert f(n=65) == f(n=-1) == f(ld=3) == f(w=-1) == ARG
    assert f(st=1028) == f(q=FAKE + 8) == f(ws=FAKE + 4) == f(w=1 << 40, ld=1 << 40) == UNS


def pages8(**kw):
    return cache8.empty(**({"pages": 4, "heads": 2, "page_size": 32, "head_dim": 64, "device": "cpu"} | kw))


def test_pages():
    c = pages8()
    assert c.k.shape == (4, 2, 32, 64) and c.k.dtype is torch.int8 and c.k_scale.shape == (4, 2, 2)
    assert pages8(dtype=torch.float8_e4m3fn).v.dtype is torch.float8_e4m3fn
    for bad in (dict(dtype=torch.uint8), dict(dtype=torch.bfloat16), dict(head_dim=80),
                dict(page_size=24), dict(page_size=8)):
        with pytest.raises(ValueError):
            pages8(**bad)
    assert c.layout("x", -1).struct.format == 1
    wide = torch.zeros(4, 2, 32, 72, dtype=torch.int8)
    for bad in (c._replace(v=c.v.view(torch.float8_e4m3fn)), c._replace(k=c.k[:3]),
                c._replace(k=wide[..., :64], v=wide[..., :64]),                 # rows of 72 bytes
                c._replace(k=c.k.transpose(2, 3)), c._replace(k_scale=c.k_scale[..., :1]),
                c._replace(v_scale=c.v_scale.double()), c._replace(v_scale=c.v_scale[:, :1]),
                cache8.Pages8(*(t[:, :, :24] for t in c[:2]), *c[2:])):
        with pytest.raises(ValueError):
            bad.layout("x", -1)
    held = c.layout("x", -1)
    assert c.layout("x", -1) is held and (held.pages, held.heads, held.page_size, held.head_dim) == (4, 2, 32, 64)
    c.k.set_(torch.zeros_like(c.k))                        # its tensors elsewhere: looked at again
    assert c.layout("x", -1).struct.k_codes == c.k.data_ptr() != held.struct.k_codes
    twin = copy.deepcopy(c)
    assert type(twin) is cache8.Pages8 and twin.layout("x", -1).struct.k_codes == twin.k.data_ptr()
    with pytest.raises(ValueError, match="cache is on"):
        c.layout("x", 0)
    with pytest.raises(RuntimeError, match="no gradient"):
        c._replace(k_scale=c.k_scale.clone().requires_grad_()).layout("x", -1)


def test_wrappers_refuse_cpu_tensors():
    c = pages8()
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    pos = torch.zeros(1, 2, dtype=torch.int64)
    table = torch.zeros(2, 1, dtype=torch.int32)
    with pytest.raises(ValueError):
        cache8.append(x, x, pos[0], c)
    with pytest.raises(ValueError):
        cache8.rotate_append(x, x, x, pos, axial.AxisPlan(torch.ones(32), [0] * 32), pos[0], c)
    with pytest.raises(ValueError):
        cache8.read(c, table, 3, 3)
    with pytest.raises(ValueError):
        cache8.attention(x[:, :, None], c, 3, table)


def test_requests_of_a_table():
    f = cache8._requests
    table = torch.zeros(3, 2, dtype=torch.int32)
    assert f("x", table, 32, 16, -1) == (3, 2, 2, None, 32)
    n = torch.ones(3, dtype=torch.int32)
    assert f("x", table, n, 16, -1)[3] == n.data_ptr()
    for bad in (table.long(), table[:, :0], table[0], table.t()):
        with pytest.raises(ValueError, match="table"):
            f("x", bad, 1, 16, -1)
    for bad in (33, -1, n[:2], n.long(), n[None]):
        with pytest.raises(ValueError, match="kv_len"):
            f("x", table, bad, 16, -1)


def test_arena_of_codes():
    for dtype in cache8.DTYPES:
        ar = PagedArena(3, 2, 6, 2, 32, 64, 64, device="cpu", dtype=dtype)
        assert ar.storage.dtype is dtype and ar.scales.shape == (3, 2, 6, 2, 2)
        codes = ar.codes(1)
        assert codes.k.data_ptr() == ar.k(1).data_ptr() and codes.v.data_ptr() == ar.v(1).data_ptr()
        assert codes.v_scale.data_ptr() == ar.scales[1, 1].data_ptr()
        assert codes.layout("x", -1).struct.format == cache8.DTYPES[dtype]
    assert PagedArena(1, 2, 6, 2, 32, 64, 64, device="cpu").scales is None
    with pytest.raises(ValueError, match="pages of"):
        PagedArena(1, 2, 6, 2, 32, 64, 64, device="cpu", dtype=torch.float16)


def test_arena_reads_bf16_pages():
    """Without a kernel: rows of each request in order, zero past its own."""
    ar = PagedArena(2, 3, 8, 2, 16, 64, 64, device="cpu")
    ar.storage.copy_(torch.randn(ar.storage.shape))
    ar.table[:] = torch.tensor([[5, 1, 0, 0], [2, 0, 0, 0], [0, 0, 0, 0]])
    ar.lens = [20, 16, 0]
    ar.kv_len.copy_(torch.tensor(ar.lens))
    for got, x in zip(ar.read(1), ar.storage[1]):
        assert got.shape == (3, 2, 20, 64)
        assert torch.equal(got[0], torch.cat((x[5], x[1, :, :4]), 1))
        assert torch.equal(got[1, :, :16], x[2]) and not got[1, :, 16:].any() and not got[2].any()
    ar.lens = [0, 0, 0]
    assert ar.read(0)[0].shape == (3, 2, 0, 64)


def test_a_cache_of_codes_plans_as_one_of_rows():
    ar = PagedArena(1, 2, 6, 2, 16, 64, 64, device="cpu", dtype=torch.int8)
    c = PagedKVCache(ar, axial.AxisPlan(torch.ones(32), [0, 1, 2, 0] * 8))
    with pytest.raises(RuntimeError, match="overflow"):
        c.begin([65, 0])
    with pytest.raises(RuntimeError, match="planned"):
        x = torch.zeros(2, 1, 2, 64, dtype=torch.bfloat16)
        c.attend(0, x, x, x, None, 1.0)
