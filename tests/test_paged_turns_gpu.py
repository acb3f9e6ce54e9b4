"""Page calls on more than one turn of their kernels' loops takes: forks beyond
512 rows and 8192 held pages, rows of more than 512 entries, copies of more
than 16384 pieces of 8 KiB, lists of more than 65536 pages."""

from __future__ import annotations

import pytest
import torch

import paged_oracle as oracle
from kda_bt16 import paged_compact, paged_copy, paged_fork, paged_free, paged_reserve
from test_paged_gpu import Pages

pytestmark = pytest.mark.gpu


def held_first(s, pages):
    """The first `pages` pages become held by someone else."""
    s.refs[:pages] = [max(1, r) for r in s.refs[:pages]]
    s.d_refs.copy_(s.ints(s.refs))


@pytest.mark.parametrize("first,spare", [(9000, 2000), (17000, 2000), (17000, 300)])
def test_forks_of_many_rows_past_many_held_pages(first, spare, gpu_device):
    s = Pages(2100, 4, first + spare, 16, gpu_device, 5, lead=(2,), page=(1, 4), used=first / (first + spare) / 2)
    rows = torch.randperm(2100, generator=torch.Generator().manual_seed(1)).tolist()
    dst, keep = rows[:1200], rows[1200:]
    paged_free(s.d_table, s.d_lens, s.d_refs, s.ints(dst))
    oracle.free(s.table, s.lens, s.refs, dst)
    s.same()
    held_first(s, first)
    src = [keep[(7 * i) % len(keep)] for i in range(1200)]
    ok = paged_fork(s.d_pool, s.d_table, s.d_lens, s.d_refs, s.ints(src), s.ints(dst))
    want = oracle.fork([s.flat()], s.table, s.lens, s.refs, src, dst, s.size)
    assert ok.tolist() == want
    assert all(want) == (spare > 300)
    s.same()


def test_long_rows(gpu_device):
    s = Pages(3, 1700, 6000, 16, gpu_device, 2, lead=(2,), page=(1, 4), used=0)
    paged_reserve(s.d_table, s.d_lens, s.d_refs, s.ints([16 * 1700, 16 * 1111 + 3, 5]), 16)
    oracle.reserve(s.table, s.lens, s.refs, [16 * 1700, 16 * 1111 + 3, 5], 16)
    s.same()
    paged_free(s.d_table, s.d_lens, s.d_refs, s.ints([2]))
    oracle.free(s.table, s.lens, s.refs, [2])
    ok = paged_fork(s.d_pool, s.d_table, s.d_lens, s.d_refs, s.ints([1]), s.ints([2]))
    assert ok.tolist() == oracle.fork([s.flat()], s.table, s.lens, s.refs, [1], [2], 16) == [True]
    s.same()
    paged_free(s.d_table, s.d_lens, s.d_refs, s.ints([0, 1]))
    oracle.free(s.table, s.lens, s.refs, [0, 1])
    s.same()


def test_copies_of_many_pieces(gpu_device):
    """Two pools: 14 parts of 1300 pages of 8 KiB + 16, 1300 pages of 32 bytes."""
    gen = torch.Generator(device=gpu_device).manual_seed(0)
    big = torch.randn(2, 7, 2700, 1, 1, 2052, generator=gen, device=gpu_device)
    small = torch.randn(2700, 1, 1, 8, generator=gen, device=gpu_device)
    order = torch.randperm(2700, generator=gen, device=gpu_device, dtype=torch.int32)
    src, dst = order[:1300].contiguous(), order[1300:2600].contiguous()
    want = [big.clone(), small.clone()]
    want[0][:, :, dst.long()] = big[:, :, src.long()]
    want[1][dst.long()] = small[src.long()]
    paged_copy([big, small], src, dst)
    assert torch.equal(big, want[0]) and torch.equal(small, want[1])


@pytest.mark.parametrize("P", [65536, 65537, 140_001])
def test_compaction_of_large_pools(P, gpu_device):
    gen = torch.Generator().manual_seed(P)
    refs = torch.randint(0, 3, (P,), generator=gen, dtype=torch.int32)
    refs[torch.rand(P, generator=gen) < 0.3] = 0
    held = torch.nonzero(refs)[:, 0].to(torch.int32)
    table = torch.full((50, 400), -1, dtype=torch.int32)
    table.view(-1)[::3] = held[torch.randint(0, len(held), (len(table.view(-1)[::3]),), generator=gen)]
    pool = torch.randn(2, P, 1, 1, 8, generator=gen)
    d_pool = pool.to(gpu_device)
    out = paged_compact(d_pool, table.to(gpu_device), refs.to(gpu_device))
    w_table, w_refs, w_live = oracle.compact([pool], [[int(x) for x in r] for r in table], refs.tolist())
    assert out[2].tolist() == [w_live]
    assert out[0].tolist() == w_table and out[1].tolist() == w_refs
    assert torch.equal(d_pool.cpu(), pool)
