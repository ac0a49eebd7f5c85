"""What the paged cache's operators refuse, before any launch (no GPU needed)."""

from __future__ import annotations

import pytest
import torch

from umic.kernels import attention, axial, paged

ARG, UNS = -1, -2
FAKE = 1 << 20  # aligned, never dereferenced: every call below returns early


@pytest.fixture(scope="module")
def lib():
    from umic import _lib

    return _lib.load()


def test_page_plan_refusals(lib):
    def f(R=4, W=8, ld=8, pages=32, page=16, tokens=4, row=0, ptrs=(FAKE,) * 12):
        return lib.umic_page_plan(*ptrs, R, W, ld, pages, page, tokens, row, None)

    def without(i):
        return tuple(None if j == i else FAKE for j in range(12))

    assert f(R=-1) == f(W=-1) == f(pages=-1) == f(tokens=-1) == f(row=-1) == f(page=0) == ARG
    assert f(ld=7) == f(W=0) == f(pages=0) == ARG
    assert f(row=2) == f(row=3, tokens=13) == ARG          # not R * row
    assert f(page=8) == f(page=24) == f(page=48) == UNS
    assert f(R=1 << 31, W=8) == f(tokens=1 << 31) == UNS
    for i in (0, 1, 4, 5, 6, 7, 8, 9, 10, 11):
        assert f(ptrs=without(i)) == ARG, i
    assert f(R=0, tokens=0, ptrs=(None,) * 12) == 0
    assert f(R=0, tokens=3) == ARG


def test_axial_refusals(lib):
    def f(T=3, Hq=4, Hk=2, D=128, axes=3, ptrs=(FAKE,) * 7, qw=None, kw=None, st=1024, sh=128):
        return lib.umic_axial_rope_bf16(*ptrs, 1.0, qw, kw, 1e-6, T, Hq, Hk, D, axes, T, 1, st, sh,
                                        st, sh, st, sh, st, sh, None)

    assert f(T=-1) == f(Hq=-1) == f(Hk=-1) == f(D=0) == f(axes=0) == ARG
    assert f(T=0, ptrs=(None,) * 7) == 0
    for i in range(7):
        assert f(ptrs=tuple(None if j == i else FAKE for j in range(7))) == ARG, i
    assert f(qw=FAKE) == f(kw=FAKE) == ARG                 # one norm without the other
    assert f(D=12) == f(D=520) == f(D=1024) == UNS
    assert f(st=1022) == f(sh=126) == UNS
    assert f(ptrs=(FAKE + 2,) + (FAKE,) * 6) == UNS
    assert f(T=1 << 40) == UNS

    def g(page=16, pages=8, slots=FAKE, v=FAKE, vp=FAKE, c=128):
        return lib.umic_axial_rope_append_bf16(
            FAKE, FAKE, v, FAKE, FAKE, vp, FAKE, FAKE, FAKE, slots, 1.0, None, None, 1e-6, 3, 4, 2,
            128, 3, 3, 1, 512, 128, 256, 128, 256, 128, 512, 128, 4096, 2048, c, pages, page, None)

    assert g(page=0) == g(pages=-1) == g(slots=None) == g(v=None) == g(vp=None) == ARG
    assert g(page=8) == g(page=20) == g(page=1 << 31) == g(c=130) == UNS


def test_cache_attention_refusals(lib):
    def f(B=2, S=1, Hq=8, Hk=2, D=128, q=FAKE, k=FAKE, v=FAKE, out=FAKE, table=None, lens=None,
          st=1024, blocks=2, rows=64, ld=0, w=0, n=64, ws=FAKE, size=1 << 40,
          scale=0.1):
        return lib.umic_cache_attention_bf16(
            q, k, v, out, table, lens, None, B, S, Hq, Hk, D, st, st, 128, st, st, 128, 16384, 8192,
            128, blocks, rows, ld, w, n, 1, scale, None, ws, size, None)

    assert f(B=-1) == f(S=-1) == f(Hq=-1) == f(Hk=-1) == f(D=0) == f(rows=-1) == f(size=-1) == ARG
    assert f(B=0) == f(S=0) == f(Hq=0) == 0
    assert f(Hk=3) == f(Hk=0) == ARG
    assert f(q=None) == f(out=None) == f(ws=None) == f(k=None) == f(v=None) == ARG
    assert f(scale=float("inf")) == f(scale=float("nan")) == f(scale=-3e38) == ARG
    assert f(blocks=3) == ARG                              # contiguous: one block a request
    assert f(n=65) == f(n=-1) == ARG                       # past the cache
    assert f(table=FAKE, w=4, ld=3) == f(table=FAKE, w=-1) == ARG
    assert f(D=80) == f(D=96) == f(D=512) == f(st=1028) == f(q=FAKE + 8) == f(ws=FAKE + 4) == UNS
    for rows in (8, 24, 40):
        assert f(table=FAKE, w=4, ld=4, rows=rows) == UNS
    assert f(table=FAKE, w=1 << 40, ld=1 << 40) == UNS
    for args in ((0, 8, 2, 128), (1, 8, 3, 128), (1, 8, 0, 128), (1, 8, 2, 80), (-1, 8, 2, 128)):
        assert lib.umic_cache_attention_workspace_bytes(*args) == 0


def test_wrappers_refuse_cpu_tensors():
    x = torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    plan = axial.AxisPlan(torch.ones(32), [0] * 32)
    pos = torch.zeros(1, 2, dtype=torch.int64)
    with pytest.raises(ValueError):
        attention.cache_attention(x, x, x, 1)
    with pytest.raises(ValueError):
        axial.rotate(x[:, :, 0], x[:, :, 0], pos, plan)
    with pytest.raises(ValueError):
        axial.rotate_append(x[:, :, 0], x[:, :, 0], x[:, :, 0], pos, plan, pos[0], x, x)
    with pytest.raises(ValueError):
        paged.plan_pages(i, i, i.view(2, 1), i, torch.zeros(4, dtype=torch.int32), 16, 2)


def test_axis_plans():
    inv = torch.tensor([1.0, 0.5, 0.25, 0.125])
    p = axial.AxisPlan(inv, [0, 1, 2, 0])
    assert p.head_dim == 8 and p.axes == 3
    # 2^64 / (2 pi), from the digits of 1 / (2 pi) = 0.15915494309189533576888376337251436203445965
    unit = 15915494309189533576888376337251436203445965 * 2 ** 64 // 10 ** 44
    for f, t in zip((0, 1, 2, 3), p.turn.tolist()):
        assert abs((t % 2 ** 64) - (unit >> f)) <= 1
    back = axial.AxisPlan(-inv, [0] * 4).turn.tolist()
    assert all((a + b) % 2 ** 64 == 0 for a, b in zip(p.turn.tolist(), back))
    for bad in (torch.tensor([1.0, float("nan")]), torch.tensor([float("inf"), 1.0]),
                torch.zeros(0), torch.ones(3), torch.ones(2, 1)):
        with pytest.raises(ValueError):
            axial.AxisPlan(bad, [0, 0])
    with pytest.raises(ValueError):
        axial.AxisPlan(torch.ones(2), [0, -1])
    t = axial.AxisPlan.text(128, 1e6, (24, 20, 20), device="cpu")
    assert [int((t.axis == a).sum()) for a in range(3)] == [24, 20, 20]
    assert t.axis[:7].tolist() == [0, 1, 2, 0, 1, 2, 0] and t.axis[60:].tolist() == [0] * 4
    t = axial.AxisPlan.text(128, 1e6, (16, 24, 24), interleaved=False, device="cpu")
    assert t.axis.tolist() == [0] * 16 + [1] * 24 + [2] * 24
    with pytest.raises(ValueError):
        axial.AxisPlan.text(128, 1e6, (24, 20, 21), device="cpu")
    with pytest.raises(ValueError):
        axial.AxisPlan.grid(82, device="cpu")
    g = axial.AxisPlan.grid(80, device="cpu")
    assert g.axis.tolist() == [0] * 20 + [1] * 20 and g.turn[:20].tolist() == g.turn[20:].tolist()
