"""Sequences that get shorter: tokens of a rejected draft come off seq_lens,
and the pages behind them stay the row's own."""

from __future__ import annotations

import random

import pytest
import torch

import paged_oracle as oracle
from kda_bt16 import paged_append, paged_attention, paged_compact, paged_fork, paged_free, paged_reserve
from test_paged_gpu import BF16, Pages, _tol

pytestmark = pytest.mark.gpu


def reserve(s, more):
    """In place on the lists of ``s``: a row's pages are its first entries, its
    own ones past its length are used before any free page."""
    free, at, ok = [p for p, r in enumerate(s.refs) if r == 0], 0, []
    for n, row in enumerate(s.table):
        want = -(-(s.lens[n] + max(0, more[n])) // s.size)
        if want > len(row):
            ok.append(False)
            continue
        have = -(-s.lens[n] // s.size)
        while have < want and row[have] >= 0:
            have += 1
        need = max(0, want - have)
        got = free[at:at + need]
        at += need
        ok.append(len(got) == need)
        if ok[-1]:
            for i, p in enumerate(got):
                row[have + i], s.refs[p] = p, 1
            s.lens[n] += max(0, more[n])
    return ok


def holders(s):
    """Every page has as many holders as rows that name it."""
    count = [0] * len(s.refs)
    for row in s.table:
        for p in row:
            if p >= 0:
                count[p] += 1
    assert count == s.refs


def step(s, more):
    ok = paged_reserve(s.d_table, s.d_lens, s.d_refs, s.ints(more), s.size)
    assert ok.tolist() == reserve(s, more)
    s.same(pool=False)
    holders(s)
    return ok.tolist()


def shorten(s, lens):
    s.lens = list(lens)
    s.d_lens.copy_(s.ints(s.lens))


def test_a_rejected_draft_across_a_page_edge(gpu_device):
    s = Pages(2, 4, 12, 16, gpu_device, 0, lead=(1,), page=(1, 4), used=0)
    step(s, [14, 30])
    step(s, [5, 5])  # a draft of 5: both rows go on to a page more
    assert sum(s.refs) == 5
    shorten(s, [15, 31])  # one token of it is right
    for _ in range(4):
        step(s, [5, 5])
        shorten(s, [s.lens[0] - 4, s.lens[1] - 4])
    assert sum(s.refs) == 5  # 24 and 40 tokens at most
    paged_free(s.d_table, s.d_lens, s.d_refs, s.ints([0, 1]))
    assert s.d_refs.tolist() == [0] * 12


def test_a_row_begun_again_keeps_its_pages(gpu_device):
    s = Pages(3, 40, 60, 16, gpu_device, 0, lead=(1,), page=(1, 4), used=0)
    step(s, [16 * 30, 16 * 5, 16 * 20])
    before = [list(r) for r in s.table]
    shorten(s, [0, 17, 100])
    assert step(s, [16 * 30, 16 * 8, 3]) == [True, True, True]
    assert s.table[0] == before[0] and s.table[2] == before[2] and s.table[1][:5] == before[1][:5]
    # no page left: those that a row has are enough for it
    shorten(s, [1, 1, 1])
    assert step(s, [16 * 38, 16 * 8 - 1, 16 * 20 - 1]) == [False, True, True]
    # 2 pages left of 60
    assert step(s, [0, 1, 16 * 2]) == [True, True, False]


@pytest.mark.parametrize("N,M,P,size", [(5, 9, 40, 16), (60, 12, 500, 32), (4200, 4, 9001, 16)])
def test_random_lengths(N, M, P, size, gpu_device):
    s = Pages(N, M, P, size, gpu_device, N, lead=(1,), page=(1, 4))
    rng = random.Random(N)
    for _ in range(5):
        step(s, [rng.choice([0, 1, 5, rng.randint(0, 3 * size)]) for _ in range(N)])
        shorten(s, [max(0, x - rng.choice([0, 0, 1, 4, rng.randint(0, 3 * size)])) for x in s.lens])
        rows = rng.sample(range(N), max(1, N // 6))
        paged_free(s.d_table, s.d_lens, s.d_refs, s.ints(rows))
        oracle.free(s.table, s.lens, s.refs, rows)
        s.same(pool=False)
        holders(s)


def test_forks_and_compaction_of_shortened_rows(gpu_device):
    s = Pages(4, 6, 30, 16, gpu_device, 1, lead=(2,), page=(1, 4), used=0)
    step(s, [70, 20, 0, 90])
    shorten(s, [30, 20, 0, 49])
    src, dst = [0], [2]
    ok = paged_fork(s.d_pool, s.d_table, s.d_lens, s.d_refs, s.ints(src), s.ints(dst))
    assert ok.tolist() == oracle.fork([s.flat()], s.table, s.lens, s.refs, src, dst, s.size) == [True]
    s.same()
    paged_free(s.d_table, s.d_lens, s.d_refs, s.ints([1]))
    oracle.free(s.table, s.lens, s.refs, [1])
    s.d_table, s.d_refs, live = paged_compact(s.d_pool, s.d_table, s.d_refs)
    s.table, s.refs, want = oracle.compact([s.flat()], s.table, s.refs)
    assert live.tolist() == [want]
    s.same()
    step(s, [40, 33, 20, 47])
    s.same()


def test_attention_after_a_rejected_draft(gpu_device):
    """Tokens written again at the same places of the same pages."""
    dev, size, HKV, D = gpu_device, 16, 2, 128
    gen = torch.Generator().manual_seed(0)
    kc, vc = (torch.randn(20, size, HKV, D, generator=gen).to(BF16) for _ in range(2))
    dk, dv = kc.to(dev), vc.to(dev)
    table = torch.full((2, 6), -1, dtype=torch.int32, device=dev)
    lens = torch.zeros(2, dtype=torch.int32, device=dev)
    refs = torch.zeros(20, dtype=torch.int32, device=dev)
    assert paged_reserve(table, lens, refs, torch.tensor([29, 44], dtype=torch.int32, device=dev), size).all()
    for kept in (1, 0, 4, 2, 5):
        assert paged_reserve(table, lens, refs, torch.full_like(lens, 5), size).all()
        k, v = (torch.randn(2, 5, HKV, D, generator=gen).to(BF16) for _ in range(2))
        paged_append(k.to(dev), v.to(dev), dk, dv, table, lens)
        oracle.append(k, v, kc, vc, table.cpu(), lens.cpu())
        q = torch.randn(2, 5, 4, D, generator=gen).to(BF16)
        want, _ = oracle.attention(q, kc, vc, table.cpu(), lens.cpu(), 0.1)
        o = paged_attention(q.to(dev), dk, dv, table, lens, scale=0.1)
        assert (o.double().cpu() - want).abs().max() <= _tol(BF16)
        lens -= 5 - kept
    assert int((refs != 0).sum()) == int((table >= 0).sum()) == 3 + 4
