"""What the 8-bit cache's operators refuse, before any launch (no GPU needed)."""

from __future__ import annotations

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


def test_append_refusals(lib):
    names = ("q", "k", "v", "qo", "kc", "vc", "ks", "vs", "pos", "turn", "axis", "slots")

    def f(T=3, Hq=4, Hk=2, D=128, axes=3, st=1024, c=2048, pages=8, page=16, fmt=0, qw=None, kw=None, **p):
        p = {n: FAKE for n in names} | p
        return lib.umic_cache8_append_bf16(
            *(p[n] for n in names), 1.0, qw, kw, 1e-6, T, Hq, Hk, D, axes, T, 1, st, 128, st, 128, st,
            128, st, 128, 4096, c, 128, 2, 1, pages, page, fmt, None)

    none = dict.fromkeys(names)
    assert f(T=-1) == f(Hq=-1) == f(Hk=0) == f(D=0) == f(axes=0) == f(pages=-1) == f(page=0) == ARG
    assert f(T=0, **none) == 0
    for n in names:
        if n != "turn":
            assert f(**{n: None}) == ARG, n
    assert f(turn=None) == ARG                             # q without a rotation
    assert f(turn=None, Hq=0, kw=FAKE) == f(turn=None, Hq=0, qw=FAKE) == ARG
    assert f(qw=FAKE) == f(kw=FAKE) == ARG                 # one norm without the other
    assert f(D=80) == f(D=512) == f(page=8) == f(page=24) == f(page=1 << 31) == UNS
    assert f(fmt=2) == f(fmt=-1) == f(pages=1 << 31) == f(pages=1 << 30, page=32) == UNS
    assert f(st=1020) == f(c=2056) == f(k=FAKE + 8) == f(kc=FAKE + 8) == f(qw=FAKE + 8, kw=FAKE) == UNS
    assert f(Hk=1 << 17) == f(T=1 << 40) == UNS


def test_read_refusals(lib):
    def f(B=2, Hk=2, rows=9, D=64, c=1024, pages=8, page=16, ld=4, w=4, n=9, fmt=1, lens=None,
          p=(FAKE,) * 7):
        return lib.umic_cache8_read_bf16(*p, lens, None, B, Hk, rows, D, 4096, c, 64, 2, 1, pages,
                                         page, ld, w, n, fmt, None)

    assert f(B=-1) == f(Hk=0) == f(rows=-1) == f(D=0) == f(pages=-1) == f(page=0) == f(w=-1) == ARG
    assert f(ld=3) == f(n=65) == f(n=-1) == f(pages=0) == ARG
    assert f(B=0, p=(None,) * 7) == f(rows=0, p=(None,) * 7) == 0
    for i in range(7):
        assert f(p=tuple(None if j == i else FAKE for j in range(7))) == ARG, i
    assert f(D=80) == f(page=8) == f(page=48) == f(fmt=7) == f(c=1032) == UNS
    assert f(w=1 << 40, ld=1 << 40) == f(B=1 << 21) == f(Hk=1 << 17) == f(rows=1 << 32) == UNS
    assert f(B=1 << 20, Hk=1 << 15) == UNS                 # more than a grid counts
    assert f(p=(FAKE + 8,) + (FAKE,) * 6) == f(p=(FAKE,) * 4 + (FAKE + 8, FAKE, FAKE)) == UNS


def test_attention_refusals(lib):
    def f(B=2, S=1, Hq=8, Hk=2, D=128, q=FAKE, k=FAKE, v=FAKE, ks=FAKE, vs=FAKE, out=FAKE, table=FAKE,
          lens=None, st=1024, c=8192, pages=2, page=64, ld=1, w=1, n=64, fmt=0, scale=0.1, ws=FAKE,
          size=1 << 40):
        return lib.umic_cache8_attention_bf16(
            q, k, v, ks, vs, out, table, lens, None, B, S, Hq, Hk, D, st, st, 128, st, st, 128, 16384, c,
            128, 8, 4, pages, page, ld, w, n, fmt, 1, scale, None, ws, size, None)

    assert f(B=-1) == f(S=-1) == f(Hq=-1) == f(Hk=-1) == f(D=0) == f(page=-1) == f(size=-1) == ARG
    assert f(B=0) == f(S=0) == f(Hq=0) == 0
    assert f(Hk=3) == f(Hk=0) == ARG
    assert f(q=None) == f(out=None) == f(ws=None) == f(k=None) == f(v=None) == ARG
    assert f(scale=float("inf")) == f(scale=float("nan")) == ARG
    assert f(n=65) == f(n=-1) == f(ld=0) == f(w=-1) == ARG
    assert f(D=80) == f(st=1028) == f(c=8200) == f(q=FAKE + 8) == f(k=FAKE + 8) == f(page=8) == UNS


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
    assert cache8._pages("x", c, -1)[0] == 1
    wide = torch.zeros(4, 2, 32, 72, dtype=torch.int8)
    for bad in (c._replace(v=c.v.view(torch.float8_e4m3fn)), c._replace(k=c.k[:3]),
                c._replace(k=wide[..., :64], v=wide[..., :64]),                 # rows of 72 bytes
                c._replace(k=c.k.transpose(2, 3)), c._replace(k_scale=c.k_scale[..., :1]),
                c._replace(v_scale=c.v_scale.double()), c._replace(v_scale=c.v_scale[:, :1]),
                cache8.Pages8(*(t[:, :, :24] for t in c[:2]), *c[2:])):
        with pytest.raises(ValueError):
            cache8._pages("x", bad, -1)
    with pytest.raises(ValueError, match="cache is on"):
        cache8._pages("x", c, 0)


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
        assert cache8._pages("x", codes, -1)[0] == cache8.DTYPES[dtype]
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
