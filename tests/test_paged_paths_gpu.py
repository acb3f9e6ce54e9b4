"""Every way that paged_attention's work is cut, against 64 bits with bounds
that follow the size of the outputs (paged_bounds.py).

The kernels' numbers: row tiles of 32 rows (few) or 256 (many) of one kv head;
tiles of 32 or 64 keys; 512 pieces of few rows (256 beside many); a table of at
most 768 keys is taken whole."""

from __future__ import annotations

import random

import pytest
import torch

import paged_bounds
from kda_bt16 import paged_attention
from test_paged_gpu import BF16, FP16, make

pytestmark = pytest.mark.gpu


def close(lens, T, HQ, HKV, D, page, dtype, dev, layout="token", causal=True, window=None, new=None, seed=0):
    (kc, vc), (dk, dv), table, ln, gen = make(lens, HKV, D, page, dtype, dev, layout, seed)
    cu = None if new is None else torch.tensor([0] + new, dtype=torch.int32).cumsum(0, dtype=torch.int32)
    shape = (len(lens), T, HQ, D) if new is None else (1, sum(new), HQ, D)
    q = torch.randn(shape, generator=gen).to(dtype)
    want = paged_bounds.expected(q, kc, vc, table, ln, D ** -0.5, causal, window, cu)
    o, lse = paged_attention(q.to(dev), dk, dv, table.to(dev), ln.to(dev), causal=causal, window=window,
                             cu_seqlens=None if cu is None else cu.to(dev), return_lse=True)
    assert paged_bounds.misses(o, lse, want, q, ln, D ** -0.5, cu) == []


def spread(n, lo, hi, seed=0):
    rng = random.Random(seed)
    return [rng.randint(lo, hi) for _ in range(n)]


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (FP16, 64), (BF16, 64), (FP16, 128)])
@pytest.mark.parametrize("T", [1, 4, 40, 300])
def test_long_sequences(T, D, dtype, gpu_device):
    """Few rows cut into pieces of 4 tiles, many rows into parts."""
    close([9000, 4099, 8192, 5000], T, 8, 1, D, 32, dtype, gpu_device, "head")


@pytest.mark.parametrize("causal,window", [(True, None), (True, 4200), (False, None)])
@pytest.mark.parametrize("D", [64, 128])
def test_many_rows_taken_whole(D, causal, window, gpu_device):
    """133 row tiles, more than half of 256: some go over 140 tiles of keys."""
    lens = [9000, 4099, 8192] + [5 + 3 * n % 60 for n in range(130)]
    close(lens, 5, 8, 1, D, 16, BF16, gpu_device, causal=causal, window=window)


@pytest.mark.parametrize("dtype,D,layout", [(BF16, 128, "head"), (FP16, 64, "token")])
@pytest.mark.parametrize("window", [None, 1000])
def test_few_rows_in_equal_pieces(window, dtype, D, layout, gpu_device):
    """512 row tiles, more than a quarter of the pieces: a piece is the end of
    one, whole ones and the start of another."""
    lens = spread(62, 30, 2500) + [0, 1]
    close(lens, 1, 32, 8, D, 16, dtype, gpu_device, layout, window=window)


@pytest.mark.parametrize("N,HKV,T", [(150, 1, 3), (130, 2, 1), (700, 1, 2)])
def test_few_rows_in_equal_pieces_of_more_than_64_sequences(N, HKV, T, gpu_device):
    close([0, 2000] + spread(N - 3, 1, 1100, N) + [1900], T, 4 * HKV, HKV, 64, 16, BF16, gpu_device)


@pytest.mark.parametrize("N,T", [(70, 1), (100, 5)])
def test_few_rows_filled_to_pieces_of_more_than_64_sequences(N, T, gpu_device):
    """At most 128 row tiles: each is filled up to whole pieces."""
    close([3000, 0] + spread(N - 3, 1, 900, N) + [2500], T, 4, 1, 64, 16, FP16, gpu_device)


def test_few_rows_of_more_than_32_tiles_a_wave(gpu_device):
    """Pieces of some 140 tiles: each wave's places are found more than once."""
    close(spread(64, 4200, 4700), 1, 8, 8, 64, 64, BF16, gpu_device, "head")


@pytest.mark.parametrize("N", [1, 31, 32, 33])
def test_few_rows_whole_by_four_and_eight_waves(N, gpu_device):
    """At most 768 keys; 256 row tiles run at once by eight waves each."""
    close(spread(N, 500, 768, N), 2, 16, 8, 128, 16, BF16, gpu_device)


@pytest.mark.parametrize("window", [None, 200])
def test_many_rows_longest_first(window, gpu_device):
    """320 row tiles of 40 sequences: taken whole, most keys first."""
    close(spread(39, 40, 700) + [1900], 40, 8, 8, 64, 16, BF16, gpu_device, window=window)


def test_many_rows_whole_of_more_than_64_sequences(gpu_device):
    close(spread(66, 20, 400), 36, 4, 4, 64, 16, FP16, gpu_device)


# (new tokens, lengths, kv heads): packed, of few and many rows in one launch.
# Cut where the table holds more than 768 keys (few), 512 or more for at most 128
# row tiles (many).
PACKED = {
    "few cut, many whole": ([1] * 15 + [40, 100, 1, 2, 64], spread(18, 300, 3000) + [1500, 2900], 8),
    "few whole, many cut": ([1, 40, 1, 300], [700, 760, 400, 768], 2),
    "both cut": ([1, 1, 64, 7, 500], [3000, 900, 5000, 2500, 2100], 2),
    "both whole": ([1, 3, 70], [490, 20, 480], 2),
    "most keys first": ([1] * 20 + [300, 40, 700, 64], spread(20, 300, 3000) + [2000, 900, 800, 2600], 8),
    "more than 64 sequences": ([1, 50, 3] * 30, [1500, 300, 40] * 30, 2),
}


@pytest.mark.parametrize("name", PACKED)
@pytest.mark.parametrize("window", [None, 900])
def test_packed(name, window, gpu_device):
    new, lens, HKV = PACKED[name]
    close(lens, 0, 4 * HKV, HKV, 128, 16, BF16, gpu_device, new=new, window=window)


def test_many_rows_in_parts(gpu_device):
    """One chunk of 64 tokens over 20000 keys; a prompt whose first row tiles
    see fewer tiles of keys than they have parts."""
    close([20000], 64, 4, 1, 64, 128, BF16, gpu_device)
    close([1500], 1500, 4, 1, 64, 128, BF16, gpu_device)
