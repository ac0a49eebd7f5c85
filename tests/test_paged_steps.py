"""Steps that a paged cache refuses, without a GPU: they change nothing."""

from __future__ import annotations

import types

import pytest
import torch

from umic import _lib, integrate
from umic.kernels import axial
from umic.paged_cache import PagedArena, PagedKVCache


def cache(requests=2, pages=6, max_tokens=64):
    ar = PagedArena(1, requests, pages, 2, 16, 64, max_tokens, device="cpu")
    return PagedKVCache(ar, axial.AxisPlan(torch.ones(32), [0, 1, 2, 0] * 8))


def refused(c, *args, match, error=ValueError, **kwargs):
    with pytest.raises(error, match=match):
        c.begin(*args, **kwargs)
    assert c.arena.lens == [0, 0] and c.arena.free == 6 and c.step is None
    assert c.arena.kv_len.tolist() == [0, 0] and c.arena.cursor.tolist() == [0, 6, 0, 0]


@pytest.mark.parametrize("rows", [1, 2, 4])
def test_positions_of_other_axes(rows):
    """Four rows are transformers' text positions ahead of the three axes: read as the axes they
    would turn height by time and width by height."""
    refused(cache(), 1, positions=torch.zeros(rows, 2, 1, dtype=torch.int64), match="each axis")


@pytest.mark.parametrize("positions", [torch.zeros(3, 2, 1, dtype=torch.int32),
                                       torch.zeros(3, 2, 1), torch.zeros(3, 2, dtype=torch.int64),
                                       torch.zeros(3, 2, 1, dtype=torch.int64, device="meta")])
def test_positions_of_another_kind(positions):
    """Refused before the plan: the first layer's refusal came when rows were counted that nothing
    had written."""
    refused(cache(), 1, positions=positions, match="positions")


def test_a_rotary_plan_of_another_kind():
    ar = cache().arena
    with pytest.raises(ValueError, match="rotary plan"):
        PagedKVCache(ar, axial.AxisPlan(torch.ones(64), [0, 1] * 32))
    with pytest.raises(ValueError, match="rotary plan"):
        PagedKVCache(ar, axial.AxisPlan(torch.ones(32), [0] * 32, device="meta"))


def test_steps_that_one_launch_does_not_take():
    """The attention counts its work in 32 bits, by what a request can hold."""
    f = _lib.lib().umic_cache_attention_max_requests
    assert f(1, 32, 8, 128, 131072) == 0x7fffffff // 8 // 4104
    assert f(32768, 32, 8, 128, 131072) == 63 and f(32768, 32, 8, 256, 131072) == 31
    assert f(1, 8, 2, 64, 16) == 1 << 20
    for args in ((0, 8, 2, 128, 64), (1, 8, 3, 128, 64), (1, 8, 2, 80, 64), (1, 8, 2, 128, -1),
                 (1 << 21, 8, 2, 128, 64), (1, 8, 2, 128, 1 << 31), (1 << 20, 1 << 16, 8, 64, 64)):
        assert f(*args) == 0
    c = cache(max_tokens=1 << 24)
    c.query_heads = 2
    assert f(1 << 18, 2, 2, 64, 1 << 24) == 0
    refused(c, [1 << 18, 0], match="one launch")


def test_modes_see_the_attention_that_the_kernel_would_replace():
    """fuse_cache_attention leaves a call to SDPA where a function or dispatch mode watches."""
    from torch.overrides import TorchFunctionMode
    from torch.utils._python_dispatch import TorchDispatchMode

    class Watch(TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    class Below(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    attn = torch.nn.Module()
    attn._umic_cache_attention = True
    attn.config = types.SimpleNamespace(_attn_implementation="sdpa")
    q = torch.zeros(1, 4, 1, 128, dtype=torch.bfloat16)
    ok = integrate._cache_attention_ok
    assert ok(attn, q, None, {})
    with torch.device("cpu"):
        assert ok(attn, q, None, {})
    for mode in (Watch(), Below()):
        with mode:
            assert not ok(attn, q, None, {})
    assert ok(attn, q, None, {})


@pytest.mark.parametrize("kind,ok", [("default", True), ("linear", True), ("yarn", True),
                                     ("dynamic", False), ("longrope", False)])
def test_rotary_modules_whose_frequencies_change(kind, ok):
    """A plan holds the frequencies as they are; a module that changes them later has none."""
    rot = torch.nn.Module()
    rot.inv_freq, rot.rope_type, rot.attention_scaling = torch.ones(32), kind, 1.5
    if ok:
        assert axial.AxisPlan.rotary(rot).scale == 1.5
    else:
        with pytest.raises(ValueError, match="rope type"):
            axial.AxisPlan.rotary(rot)
