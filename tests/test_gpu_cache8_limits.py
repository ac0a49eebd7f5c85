"""Calls of the 8-bit cache's operators at their limits: memory that rows share, the largest values,
reads and deals of many workgroups, prompts."""

from __future__ import annotations

import pytest
import torch

from helpers import bf16_randn
from test_gpu_cache8 import DEV, call, filled, queries
from umic.kernels import axial, cache8

pytestmark = pytest.mark.gpu


def test_rows_that_share_memory_are_read_not_written():
    cache, table, _, _ = filled("int8", [40], 2, 64, 16, seed=1)
    p = int(table[0, 1])
    thrice = cache8.Pages8(*(t[p:p + 1].expand(3, *t.shape[1:]) for t in cache))
    each, same = (torch.tensor([x], dtype=torch.int32, device=DEV) for x in ([0, 1, 2], [p, p, p]))
    for got, want in zip(cache8.read(thrice, each, 48, 48), cache8.read(cache, same, 48, 48)):
        assert torch.equal(got, want)
    q = queries(1, 1, 4, 64, 1)
    assert torch.equal(call(q, thrice, [48], each), call(q, cache, [48], same))
    x = bf16_randn(4, 2, 64, gen=torch.Generator().manual_seed(1)).to(DEV)
    at = torch.arange(4, device=DEV)
    plan = axial.AxisPlan(torch.ones(32), [0] * 32, device=DEV)
    for bad in (thrice, cache._replace(v=cache.k), cache._replace(v_scale=cache.k_scale)):
        before = [t.clone() for t in cache]
        with pytest.raises(ValueError, match="share memory"):
            cache8.append(x, x, at, bad)
        with pytest.raises(ValueError, match="share memory"):
            cache8.rotate_append(x, x, x, at[None], plan, at, bad)
        for t, was in zip(cache, before):
            assert torch.equal(t.view(torch.uint8), was.view(torch.uint8))
