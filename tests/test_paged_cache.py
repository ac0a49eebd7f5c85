"""The paged cache's host side, without a GPU: geometry, overflow, what it refuses, and what the
other caches leave to it."""

from __future__ import annotations

import pytest
import torch

from umic import UmicConfig, integrate
from umic.cache import CacheStandIn
from umic.graph import DecodeGraphRunner
from umic.kernels import axial
from umic.optimize import _plan
from umic.paged_cache import PagedArena, PagedKVCache


def cache(requests=2, pages=6, max_tokens=64):
    ar = PagedArena(1, requests, pages, 2, 16, 64, max_tokens, device="cpu")
    return PagedKVCache(ar, axial.AxisPlan(torch.ones(32), [0, 1, 2, 0] * 8))


@pytest.mark.parametrize("bad", [dict(layers=0), dict(requests=0), dict(pages=0), dict(heads=0),
                                 dict(max_tokens=0), dict(page_size=8), dict(page_size=24),
                                 dict(head_dim=80)])
def test_geometry(bad):
    args = dict(layers=1, requests=2, pages=4, heads=2, page_size=16, head_dim=64, max_tokens=50)
    assert PagedArena(**args, device="cpu").max_tokens == 64
    with pytest.raises(ValueError):
        PagedArena(**{**args, **bad}, device="cpu")


def test_a_step_that_does_not_fit_changes_nothing():
    c = cache()
    for new, keep, error in (([65, 0], None, RuntimeError), ([64, 33], None, RuntimeError),
                             ([1], None, ValueError), ([1, -1], None, ValueError),
                             ([1, 1], [0], ValueError)):
        with pytest.raises(error):
            c.begin(new, keep=keep)
        assert c.arena.lens == [0, 0] and c.arena.free == 6 and c.step is None
    with pytest.raises(ValueError):
        c.begin(2, positions=torch.zeros(3, 2, 1, dtype=torch.int64))
    with pytest.raises(ValueError):  # the plan itself runs on the GPU
        c.begin(1)
    assert c.arena.lens == [0, 0] and c.arena.free == 6 and c.step is None


def test_what_it_refuses():
    c = cache()
    x = torch.zeros(2, 1, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        c.attend(0, x, x, x, None, 1.0)    # no step begun
    with pytest.raises(RuntimeError):
        c.update(x, x, 0)
    with pytest.raises(RuntimeError):
        c.crop(3)
    for call in (c.reorder_cache, c.batch_select_indices, c.batch_repeat_interleave):
        with pytest.raises(RuntimeError):
            call(torch.tensor([1, 0]))
    with pytest.raises(ValueError, match="attention_mask"):
        integrate._paged_attention(torch.nn.Module(), x, torch.ones(2, 1), c, None)
    assert c.get_seq_length() == 0 and c.get_mask_sizes(5, 0) == (5, 0)
    assert c.get_max_length() == 64


def test_other_caches_leave_it_alone():
    c = cache()
    assert not CacheStandIn.convertible(c)

    class VLM(torch.nn.Module):
        def forward(self, **kwargs):
            return kwargs["past_key_values"]

    runner = DecodeGraphRunner(VLM())
    c._before = [3, 3]
    assert not runner._is_step((), {"input_ids": torch.zeros(1, 1, dtype=torch.long),
                                    "past_key_values": c})


def test_cache_attention_is_off_unless_asked_for():
    keys = ("lm_cache_attention", "expert_cache_attention")
    wanted = {key: want for want, _, key, _ in _plan(integrate)}
    assert not any(wanted[k](UmicConfig()) for k in keys)
    assert all(wanted[k](UmicConfig(cache_attention=True)) for k in keys)
    assert not any(wanted[k](UmicConfig(cache_attention=True, text_rope_fusion=False))
                   for k in keys)
    assert not wanted[keys[1]](UmicConfig(cache_attention=True, flow_cache=False))
