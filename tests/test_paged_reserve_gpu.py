"""paged_reserve over more sequences, pages and requests than one turn of its
loops takes."""

from __future__ import annotations

import pytest
import torch

import paged_oracle as oracle
from kda_bt16 import paged_reserve
from test_paged_gpu import Pages

pytestmark = pytest.mark.gpu


def reserve(s, more):
    ok = paged_reserve(s.d_table, s.d_lens, s.d_refs, s.ints(more), s.size)
    want = oracle.reserve(s.table, s.lens, s.refs, more, s.size)
    assert ok.tolist() == want
    s.same(pool=False)
    return want


def pages(N, M, P, seed, dev, used=0.0):
    return Pages(N, M, P, 16, dev, seed, lead=(1,), page=(1, 4), used=used)


def test_pages_run_out_among_the_first_4096_sequences(gpu_device):
    """Row 0 asks for more than there is and gives back what it got: later
    sequences get none of it, on whichever side of 4096 they are."""
    s = pages(4100, 6, 3, 0, gpu_device)
    more = [0] * 4100
    more[0], more[1], more[4095], more[4096], more[4099] = 80, 1, 1, 1, 33
    assert reserve(s, more) == [n not in (0, 1, 4095, 4096, 4099) for n in range(4100)]


@pytest.mark.parametrize("P", [700, 4000, 9000, 17000, 40000])
@pytest.mark.parametrize("N,seed", [(4097, 1), (8200, 2), (9000, 3)])
def test_thousands_of_sequences(N, P, seed, gpu_device):
    """Pages run out in the first 4096, the second, the third, or not at all."""
    s = pages(N, 5, P, seed, gpu_device, used=0.3)
    gen = torch.Generator().manual_seed(seed)
    for step in range(2):
        more = torch.randint(-3, 60, (N,), generator=gen)
        more[torch.rand(N, generator=gen) < 0.3] = 0
        reserve(s, more.tolist())


@pytest.mark.parametrize("P", [3000, 9001, 30000])
def test_more_than_4096_pages_for_few_sequences(P, gpu_device):
    s = pages(5, 5000, P, 7, gpu_device, used=0.4)
    reserve(s, [16 * 1000, 3, 16 * 3000 + 5, 16 * 4100, 1])


# Tables of 11 GB and 19 GB; requests for more than 2^31 pages in all, and for more than 2^32.
@pytest.mark.parametrize("N,M", [(4096, 5 << 17), (70, (1 << 26) - 1)])
def test_requests_past_32_bits(N, M, gpu_device):
    """More pages wanted than 32 bits count: the first two rows get theirs, the
    third what is left and gives it back, the others none."""
    P, size, dev = 100, 16, gpu_device
    table = torch.full((N, M), -1, dtype=torch.int32, device=dev)
    lens = torch.zeros(N, dtype=torch.int32, device=dev)
    refs = torch.zeros(P, dtype=torch.int32, device=dev)
    refs[::2] = 1
    more = torch.full((N,), M * size, dtype=torch.int32, device=dev)
    more[:2] = torch.tensor([1, 33], dtype=torch.int32)
    more[-2:] = torch.tensor([0, 8 * size], dtype=torch.int32)
    ok = paged_reserve(table, lens, refs, more, size)
    assert ok.tolist() == [True, True] + [False] * (N - 4) + [True, False]
    assert lens.tolist() == [1, 33] + [0] * (N - 2)
    assert refs.tolist() == [int(p % 2 == 0 or p < 8) for p in range(P)]
    assert table[0, :2].tolist() == [1, -1] and table[1, :4].tolist() == [3, 5, 7, -1]
    held = [n for n in range(N) if bool((table[n] >= 0).any())]
    assert held == [0, 1]
