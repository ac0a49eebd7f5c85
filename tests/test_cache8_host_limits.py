"""Limits of the 8-bit cache's entry points that a call meets before any launch (no GPU needed)."""

from __future__ import annotations


from test_cache8_host import FAKE, UNS, lib, struct  # noqa: F401


def test_tokens_of_a_call(lib):  # noqa: F811
    """Distances between tokens are 32-bit numbers."""
    at, keep = struct()
    for T in (1 << 31, 1 << 40):
        assert lib.umic_cache8_append_bf16(at, None, FAKE, FAKE, None, None, None, None, FAKE, 1.0, None,
                                           None, 0.0, T, 0, 0, 0, 0, *[1024, 64] * 3, None) == UNS
