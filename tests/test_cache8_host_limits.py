"""Limits of the 8-bit cache's entry points that a call meets before any launch (no GPU needed)."""

from __future__ import annotations


import pytest
import torch

from test_cache8_host import FAKE, UNS, lib, pages8, struct  # noqa: F401
from umic.kernels import cache8
from umic.paged_cache import PagedArena


def test_tokens_of_a_call(lib):  # noqa: F811
    """Distances between tokens are 32-bit numbers."""
    at, keep = struct()
    for T in (1 << 31, 1 << 40):
        assert lib.umic_cache8_append_bf16(at, None, FAKE, FAKE, None, None, None, None, FAKE, 1.0, None,
                                           None, 0.0, T, 0, 0, 0, 0, *[1024, 64] * 3, None) == UNS


def test_rows_that_share_memory():
    """Expanded codes or scales, rows that overlap, keys that are the values: looked at, and not
    for an append.  Layouts of any order, gaps, and keys between values are."""
    c = pages8()
    apart = lambda **kw: c._replace(**kw).layout("x", -1).apart  # noqa: E731
    assert apart()
    lap = torch.zeros(4 * 2 * 32 * 64, dtype=torch.int8).as_strided(c.k.shape, (4096, 2048, 48, 1))
    for bad in (dict(k=c.k[:1].expand(4, -1, -1, -1), v=c.v[:1].expand(4, -1, -1, -1)),
                dict(k=c.k[:, :1].expand(-1, 2, -1, -1), v=c.v[:, :1].expand(-1, 2, -1, -1)),
                dict(k_scale=c.k_scale[:1].expand(4, -1, -1), v_scale=c.v_scale[:1].expand(4, -1, -1)),
                dict(v=c.k), dict(v_scale=c.k_scale), dict(k=lap, v=torch.zeros_like(lap).as_strided(lap.shape, lap.stride()))):
        assert not apart(**bad), {k: (v.shape, v.stride()) for k, v in bad.items()}
    both = torch.zeros(4, 2, 32, 2, 64, dtype=torch.int8)           # a row of k, one of v
    assert apart(k=both[..., 0, :], v=both[..., 1, :])
    turned = torch.zeros(2, 4, 32, 2, 80, dtype=torch.int8)[..., :64]  # rows of heads, with gaps
    assert apart(k=turned[0].transpose(1, 2), v=turned[1].transpose(1, 2))
    scales = torch.zeros(4, 2, 2, 2)
    assert apart(k_scale=scales[..., 0, :], v_scale=scales[..., 1, :])
    pool = torch.zeros(9, 2, 32, 64, dtype=torch.int8)
    assert apart(k=pool[:4], v=pool[4:8]) and not apart(k=pool[:4], v=pool[3:7])
    assert cache8.empty(0, 2, 16, 64, torch.int8, "cpu").layout("x", -1).apart
    one = cache8.empty(1, 1, 16, 64, torch.int8, "cpu")
    assert one.layout("x", -1).apart and not one._replace(v=one.k).layout("x", -1).apart


def test_codes_of_an_arena_of_rows():
    ar = PagedArena(2, 2, 6, 2, 32, 64, 64, device="cpu")
    with pytest.raises(ValueError, match="bf16 rows"):
        ar.codes(0)
