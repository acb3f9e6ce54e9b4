"""The bounds of paged_bounds.py on the CPU: results that are rounded as the
kernels round them keep them, and one wrong tile of keys or values, at any
place of a long sequence, does not."""

from __future__ import annotations

import pytest
import torch

import paged_bounds
from test_paged_gpu import BF16, FP16, _tol, make

CPU = torch.device("cpu")


def case(L, D, dtype, T=5, HQ=8, HKV=1):
    (kc, vc), _, table, ln, gen = make([L], HKV, D, 16, dtype, CPU)
    q = torch.randn(1, T, HQ, D, generator=gen).to(dtype)
    return q, kc, vc, table, ln


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("L,D", [(5, 64), (64, 128), (1000, 128), (9000, 128), (9000, 64)])
def test_rounding_keeps_the_bounds(L, D, dtype):
    q, kc, vc, table, ln = case(L, D, dtype)
    want = paged_bounds.expected(q, kc, vc, table, ln, D ** -0.5)
    o = paged_bounds.rounded(q, kc, vc, table, ln, D ** -0.5)
    assert paged_bounds.misses(o, want[1], want, q, ln, D ** -0.5) == []


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("which", ["keys", "values"])
@pytest.mark.parametrize("tile,keys", [(0, 64), (64, 64), (139, 64), (128, 32), (140, 32), (255, 32)])
def test_one_wrong_tile_is_seen(tile, keys, which, dtype):
    """Tile `tile` of `keys` keys holds the one before (the first: the one
    after): a place in a ring or a table entry read a tile late."""
    L, D = 9000, 128
    q, kc, vc, table, ln = case(L, D, dtype)
    want = paged_bounds.expected(q, kc, vc, table, ln, D ** -0.5)
    pages = keys // 16
    to, src = tile * pages, (tile - 1 if tile else 1) * pages
    c = (kc if which == "keys" else vc).clone()
    for i in range(pages):
        c[int(table[0, to + i])] = c[int(table[0, src + i])]
    caches = (c, vc) if which == "keys" else (kc, c)
    bad = paged_bounds.expected(q, *caches, table, ln, D ** -0.5)
    found = paged_bounds.misses(bad[0], bad[1], want, q, ln, D ** -0.5)
    assert any("root mean square" in x for x in found), found
    if which == "values":
        # (a bound that does not follow o's size sees nothing of it)
        assert (bad[0] - want[0]).abs().max() <= _tol(BF16)
