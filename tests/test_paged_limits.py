"""Sizes at which the paged cache's kernels would leave 32 bits: refused
before any launch (CPU only)."""

from __future__ import annotations

import ctypes

import pytest

from kda_bt16 import _hip
from test_paged_capi import fake_pointers, pages


@fake_pointers
@pytest.mark.parametrize("name", ["reserve", "free", "fork", "compact"])
def test_page_counts_near_the_end_of_32_bits(name):
    """The kernels step over the counts 16384 at a time and compare where they
    are with the number of pages: up to there has to be a number of 32 bits."""
    f = getattr(_hip.lib(), f"kda_pages_{name}_hip")
    for P in ((1 << 31) - 1, (1 << 31) - 16384, (1 << 31) - (1 << 16)):
        assert f(ctypes.byref(pages(P=P, workspace_bytes=1 << 40)), None) == -2, P
