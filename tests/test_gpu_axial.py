"""Rotary positions of several axes (umic_axial_rope_bf16 and its append) against the formula
in 64 bits, within one bf16 rounding; pages and rows that no slot names keep their bits."""

from __future__ import annotations

import pytest
import torch

import paged_reference as ref
from helpers import bf16_randn
from umic.kernels import axial

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(T, Hq, Hk, D, axes=3, seed=0, hi=40000):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (bf16_randn(T, h, D, gen=g).to(DEV) for h in (Hq, Hk, Hk))
    inv = (1e4 ** (-torch.arange(D // 2) / (D // 2))).float()
    axis = torch.randint(0, axes, (D // 2,), generator=g)
    axis[0] = axes - 1
    pos = torch.randint(-hi, hi, (axes, T), generator=g)
    w = tuple(bf16_randn(D, scale=0.1, shift=1.0, gen=g).to(DEV) for _ in range(2))
    return q, k, v, inv, axis, pos.to(DEV), w


@pytest.mark.parametrize("T", [1, 3, 4, 5, 129])
@pytest.mark.parametrize("Hq,Hk,D", [(32, 8, 128), (8, 2, 64), (4, 4, 80), (3, 1, 72), (2, 1, 256),
                                     (5, 5, 96), (1, 1, 512), (14, 2, 8)])
@pytest.mark.parametrize("norm", [False, True])
def test_rotate(T, Hq, Hk, D, norm):
    q, k, _, inv, axis, pos, w = make(T, Hq, Hk, D, seed=T + D)
    plan = axial.AxisPlan(inv, axis, 1.25, DEV)
    qo, ko = axial.rotate(q, k, pos, plan, (*w, 1e-5) if norm else None)
    for got, x, nw in ((qo, q, w[0]), (ko, k, w[1])):
        want, size = ref.rotate(x, pos, inv, axis, nw if norm else None, 1e-5, 1.25)
        ref.check_rotated(got, want, size, norm)


def test_far_positions_turn_exactly():
    """Positions whose fp32 products with a frequency have no fraction left."""
    inv = torch.tensor([1.0, 0.7310586, 1e-3, 3.0])
    pos = torch.tensor([[2 ** 28 + 1, -(2 ** 28) - 3, 2 ** 27 + 12345, 0]], device=DEV)
    q = bf16_randn(4, 2, 8, gen=torch.Generator().manual_seed(1)).to(DEV)
    plan = axial.AxisPlan(inv, [0] * 4, device=DEV)
    got, _ = axial.rotate(q, q, pos, plan)
    # 28-bit positions times 24-bit frequencies are exact in 53 bits, as ref takes them
    want, size = ref.rotate(q, pos, inv, [0] * 4)
    ref.check_rotated(got, want, size)


def test_packed_projection_and_broadcast_positions():
    """q and k of a packed projection, positions of one axis shown as three, token-major ones."""
    T, H, D = 37, 4, 64
    g = torch.Generator().manual_seed(2)
    qkv = bf16_randn(T, 3, H, D, gen=g).to(DEV)
    inv = (1e4 ** (-torch.arange(D // 2) / (D // 2))).float()
    plan = axial.AxisPlan(inv, torch.arange(D // 2) % 3, device=DEV)
    one = torch.randint(0, 500, (T,), generator=g).to(DEV)
    major = torch.randint(0, 500, (T, 3), generator=g).to(DEV).t()
    for pos in (one.expand(3, T), major):
        got = axial.rotate(qkv[:, 0], qkv[:, 1], pos, plan)
        for x, o in zip((qkv[:, 0], qkv[:, 1]), got):
            ref.check_rotated(o, *ref.rotate(x, pos, inv, torch.arange(D // 2) % 3))


def test_unaligned_rows_are_copied():
    x = bf16_randn(6, 2, 65, gen=torch.Generator().manual_seed(3)).to(DEV)[..., 1:]
    inv = torch.ones(32)
    pos = torch.arange(6, device=DEV)[None]
    got, _ = axial.rotate(x, x, pos, axial.AxisPlan(inv, [0] * 32, device=DEV))
    ref.check_rotated(got, *ref.rotate(x, pos, inv, [0] * 32))


@pytest.mark.parametrize("page,Hq,Hk,D,norm", [(16, 32, 8, 128, True), (64, 8, 2, 64, False),
                                               (32, 2, 2, 80, True), (16, 3, 1, 72, False)])
def test_append(page, Hq, Hk, D, norm):
    T, pages = 53, 9
    q, k, v, inv, axis, pos, w = make(T, Hq, Hk, D, seed=page)
    plan = axial.AxisPlan(inv, axis, device=DEV)
    g = torch.Generator().manual_seed(5)
    slots = torch.randperm(pages * page, generator=g)[:T]
    slots[3], slots[10], slots[52] = -1, pages * page, -(1 << 40)  # written nowhere
    store = bf16_randn(2, pages, Hk, page, D, gen=g).to(DEV)
    before = store.clone()
    got = axial.rotate_append(q, k, v, pos, plan, slots.to(DEV), store[0], store[1],
                              (*w, 1e-6) if norm else None)
    ref.check_rotated(got, *ref.rotate(q, pos, inv, axis, w[0] if norm else None), norm)
    want, size = ref.rotate(k, pos, inv, axis, w[1] if norm else None)
    flat = store.transpose(2, 3).reshape(2, pages * page, Hk, D)  # [2, slot, Hk, D]
    was = before.transpose(2, 3).reshape(2, pages * page, Hk, D)
    real = (slots >= 0) & (slots < pages * page)
    ref.check_rotated(flat[0][slots[real].to(DEV)], want[real], size[real], norm)
    assert torch.equal(flat[1][slots[real].to(DEV)], v[real.to(DEV)])
    rest = torch.ones(pages * page, dtype=torch.bool)
    rest[slots[real]] = False
    assert torch.equal(flat[:, rest.to(DEV)], was[:, rest.to(DEV)])


def test_plan_of_a_text_rotary_module():
    """The plan turns as the tables of transformers' own rotary module do (its cos and sin are
    fp32 products of positions below 2^11: 2^-13 of a radian; then bf16)."""
    from helpers import qwen3_decoder_layer

    _, rot = qwen3_decoder_layer()
    T = 70
    pos = torch.randint(0, 2000, (3, T), generator=torch.Generator().manual_seed(4)).to(DEV)
    x = torch.zeros(T, 1, 128, dtype=torch.bfloat16, device=DEV)
    x[..., :64] = 1  # first halves one, second zero: the output is (cos, sin)
    got, _ = axial.rotate(x, x, pos, axial.AxisPlan.rotary(rot))
    cos, sin = rot(x[None, :, 0].float(), pos[:, None])
    want = torch.cat((cos[0, :, :64], sin[0, :, :64]), -1)
    assert (got[:, 0].float() - want).abs().max() <= 2.0 ** -8 + 2.0 ** -12


def test_grid_plan():
    side, D = 6, 80
    pos = torch.stack((torch.arange(36) // side, torch.arange(36) % side)).to(DEV)
    x = bf16_randn(36, 2, D, gen=torch.Generator().manual_seed(6)).to(DEV)
    inv = (1.0 / 1e4 ** (torch.arange(0, 40, 2, dtype=torch.float32) / 40)).repeat(2)
    got, _ = axial.rotate(x, x, pos, axial.AxisPlan.grid(D))
    ref.check_rotated(got, *ref.rotate(x, pos, inv, [0] * 20 + [1] * 20))


def test_stream_and_capture():
    q, k, v, inv, axis, pos, w = make(9, 8, 2, 128, seed=8)
    plan = axial.AxisPlan(inv, axis, device=DEV)
    store = torch.zeros(2, 2, 2, 16, 128, dtype=torch.bfloat16, device=DEV)
    slots = torch.arange(9, device=DEV)
    want = axial.rotate_append(q, k, v, pos, plan, slots, store[0], store[1], (*w, 1e-6))
    kept = store.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        store.zero_()
        got = axial.rotate_append(q, k, v, pos, plan, slots, store[0], store[1], (*w, 1e-6))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(store, kept)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = axial.rotate_append(q, k, v, pos, plan, slots, store[0], store[1], (*w, 1e-6))
    for step in range(3):
        pos.add_(1)
        slots.add_(1)
        want = axial.rotate_append(q, k, v, pos, plan, slots, kept[0], kept[1], (*w, 1e-6))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(store, kept)
