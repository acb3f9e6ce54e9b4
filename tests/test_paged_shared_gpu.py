"""Attention of sequences in groups that share their first tokens, on the GPU
against its definition in 64 bits (every sequence by itself); bounds as for
paged_attention (tests/paged_bounds.py)."""

from __future__ import annotations

import pytest
import torch

from kda_bt16 import (
    paged_append,
    paged_attention,
    paged_attention_shared,
    paged_fork,
    paged_free,
    paged_reserve,
)
from paged_bounds import misses
from paged_seen_oracle import attention, caches, held_tokens, on_device, tables

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def make(groups, own, page, HKV, D, dtype, gen, layout="token", before=0, after=0, wide=True):
    """``groups``: (shared tokens, sequences) each; ``own(n)``: sequence n's
    tokens behind them; ``before`` and ``after``: rows of no group at the ends.
    ``wide``: a table whose rows have room for 256 MB of keys and values (those of
    less are worked on one by one).  Caches, table, lengths and the groups'
    tensors, on the CPU."""
    lens, starts, shared, members = [], [before], [], []
    lens += [own(n) for n in range(before)]
    for tokens, count in groups:
        members.append(range(len(lens), len(lens) + count))
        lens += [tokens + own(len(lens) + i) for i in range(count)]
        starts.append(len(lens))
        shared.append(tokens)
    lens += [own(len(lens) + i) for i in range(after)]
    table, P = tables(lens, page, gen, -(-(256 << 20) // (len(lens) * HKV * D * 4 * page)) if wide else 0)
    for (tokens, _), rows in zip(groups, members):
        for n in rows:
            table[n, :tokens // page] = table[rows[0], :tokens // page]
    kc, vc = caches(table, P, HKV, D, page, dtype, held_tokens(table, P, lens, page), gen, layout)
    for (tokens, _), rows in zip(groups, members):
        if tokens % page:  # the last partial page: copies
            at = [int(table[n, tokens // page]) for n in rows]
            for c in (kc, vc):
                for a in at[1:]:
                    c[a, :tokens % page] = c[at[0], :tokens % page]
    i32 = torch.int32
    return kc, vc, table, torch.tensor(lens, dtype=i32), torch.tensor(starts, dtype=i32), torch.tensor(shared, dtype=i32)


def compare(dev, q, kc, vc, table, lens, starts, shared, cu=None, want=None):
    scale = q.shape[-1] ** -0.5
    if want is None:
        want = attention(q, kc, vc, table, lens, scale, lambda pos, j: j <= pos, cu)
    o, lse = paged_attention_shared(q.to(dev), on_device(kc, dev), on_device(vc, dev), table.to(dev), lens.to(dev),
                                    starts.to(dev), shared.to(dev), cu_seqlens=None if cu is None else cu.to(dev),
                                    return_lse=True)
    assert o.shape == q.shape and o.dtype == q.dtype
    wrong = misses(o, lse, want, q, lens.tolist(), scale, cu)
    assert not wrong, wrong
    return o, lse


def check(dev, groups, own=None, T=1, HQ=4, HKV=2, D=128, page=16, dtype=BF16, layout="token", new=None, before=0, after=0,
          seed=0, wide=True, cu_dtype=torch.int32):
    gen = torch.Generator().manual_seed(seed)
    new_of = (lambda n: T) if new is None else (lambda n: new[n])
    own = own or (lambda n: new_of(n) + (37 * n) % 61)
    kc, vc, table, lens, starts, shared = make(groups, own, page, HKV, D, dtype, gen, layout, before, after, wide)
    cu = None if new is None else torch.tensor([0] + new).cumsum(0).to(cu_dtype)
    q = torch.randn(*((len(lens), T) if new is None else (1, sum(new))), HQ, D, generator=gen).to(dtype)
    return compare(dev, q, kc, vc, table, lens, starts, shared, cu)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("shared", [1, 15, 16, 31, 32, 33, 64, 100, 700, 3001])
def test_decode_prefixes(dtype, D, shared, gpu_device):
    check(gpu_device, [(shared, 5)], D=D, dtype=dtype)


@pytest.mark.parametrize("count", [1, 2, 3, 8, 16, 17, 33, 64, 130])
@pytest.mark.parametrize("T", [1, 3])
def test_group_sizes(count, T, gpu_device):
    check(gpu_device, [(333, count)], T=T)


@pytest.mark.parametrize("HQ,HKV", [(1, 1), (3, 1), (10, 2), (32, 8), (40, 1), (16, 16), (70, 2), (127, 1), (130, 1)])
@pytest.mark.parametrize("T", [1, 4])
def test_heads(HQ, HKV, T, gpu_device):
    check(gpu_device, [(200, 6), (75, 3)], T=T, HQ=HQ, HKV=HKV)


@pytest.mark.parametrize("T", [2, 8, 16, 17, 40, 100, 127, 128, 200])
def test_new_tokens(T, gpu_device):
    """Sequences of few rows, of many, and (from 128 on) of whole row tiles,
    which are worked on one by one."""
    check(gpu_device, [(300, 3), (130, 2)], T=T)


@pytest.mark.parametrize("T,HQ,HKV,D", [(65, 4, 2, 64), (100, 4, 2, 128), (127, 4, 2, 64), (33, 8, 2, 128), (60, 8, 2, 64), (1, 258, 2, 64)])
def test_dense_rows_past_a_row_tile_go_one_by_one(T, HQ, HKV, D, gpu_device):
    """From 129 rows a sequence on none shares: paged_attention's own launches."""
    d, gen = gpu_device, torch.Generator().manual_seed(17)
    kc, vc, table, lens, starts, shared = make([(300, 3), (130, 2)], lambda n: T + 9 * n, 16, HKV, D, BF16, gen)
    q = torch.randn(5, T, HQ, D, generator=gen).to(BF16)
    o, lse = compare(d, q, kc, vc, table, lens, starts, shared)
    want, want_lse = paged_attention(q.to(d), kc.to(d), vc.to(d), table.to(d), lens.to(d), return_lse=True)
    assert torch.equal(o, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("T,HQ,HKV,D,dtype", [(65, 4, 2, 64, BF16), (40, 8, 2, 128, FP16), (1, 130, 1, 64, BF16), (127, 2, 1, 64, FP16)])
def test_dense_rows_past_a_row_tile_in_finer_parts(T, HQ, HKV, D, dtype, gpu_device):
    """65 to 128 row tiles of 256: by the plan, in row tiles of 128, none shared."""
    N = 70 // HKV
    check(gpu_device, [(300, N - 12), (130, 12)], T=T, HQ=HQ, HKV=HKV, D=D, dtype=dtype)


@pytest.mark.parametrize("T,HQ,HKV,D", [(1, 16, 8, 128), (4, 16, 8, 128), (5, 24, 8, 128), (1, 16, 16, 64)])
def test_rows_that_one_launch_takes_whole_go_one_by_one(T, HQ, HKV, D, gpu_device):
    """Rows of up to 768 keys: paged_attention's own launch, whatever they hold in
    all (here 256 MB and more)."""
    d, gen = gpu_device, torch.Generator().manual_seed(18)
    N = 1024 // HKV
    kc, vc, table, lens, starts, shared = make([(600, N - 10), (130, 10)], lambda n: T + n % 9, 16, HKV, D, BF16, gen, wide=False)
    table = torch.cat([table, torch.full((N, 48 - table.shape[1]), -1, dtype=torch.int32)], 1)
    q = torch.randn(N, T, HQ, D, generator=gen).to(BF16)
    o, lse = compare(d, q, kc, vc, table, lens, starts, shared)
    want, want_lse = paged_attention(q.to(d), kc.to(d), vc.to(d), table.to(d), lens.to(d), return_lse=True)
    assert torch.equal(o, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("page", [16, 64, 1024])
@pytest.mark.parametrize("layout", ["token", "head"])
def test_pages(page, layout, gpu_device):
    check(gpu_device, [(1500, 4), (1024, 3), (17, 2)], page=page, layout=layout)
    check(gpu_device, [(1500, 4), (1024, 3), (17, 2)], page=page, layout=layout, T=20)


def test_narrow_tables(gpu_device):
    for T in (1, 20):
        check(gpu_device, [(300, 4), (90, 3)], T=T, wide=False, after=1)


def test_several_groups_and_rows_of_none(gpu_device):
    check(gpu_device, [(64, 3), (0, 2), (500, 1), (90, 4)], before=3, after=2)
    check(gpu_device, [(64, 3), (0, 2), (500, 1), (90, 4)], before=3, after=2, T=9)


@pytest.mark.parametrize("cu_dtype", [torch.int32, torch.int64])
def test_packed(cu_dtype, gpu_device):
    new = [1, 0, 3, 1, 40, 1, 1, 2, 100, 1]
    check(gpu_device, [(200, 4), (333, 4)], new=new, before=1, after=1, cu_dtype=cu_dtype, own=lambda n: new[n] + 3 * n)


def test_packed_with_a_chunk_in_a_group(gpu_device):
    """A sequence of whole row tiles in a group: all of the group by themselves;
    in a group of its own it leaves the others theirs."""
    new = [1, 1, 300, 1, 1, 1]
    check(gpu_device, [(200, 6)], new=new)
    check(gpu_device, [(200, 2), (150, 1), (200, 3)], new=new)


@pytest.mark.parametrize("new", [[1] * 63 + [60], [60] + [1] * 63, [8] * 64, [63] + [1] * 20 + [200] + [1] * 42])
def test_packed_uneven_rows_are_joined(new, gpu_device):
    """A few sequences with most of the rows, and rows enough for every
    work-group of the join to take more than one pass."""
    check(gpu_device, [(400, 64)], new=new, HQ=32, HKV=8, own=lambda n: new[n] + 20)


@pytest.mark.parametrize("dtype,D,HQ,HKV", [(FP16, 64, 128, 32), (BF16, 128, 128, 32), (BF16, 64, 96, 16)])
@pytest.mark.parametrize("own", [20, 3000])
def test_packed_long_chunks_beside_a_group(own, dtype, D, HQ, HKV, gpu_device):
    """Row tiles enough for several rounds: chunks in row tiles of 256, whose
    last may be of few rows, whole and (those of one far longer sequence) cut."""
    new = [400, 1, 60, 33, 1, 290, 64, 1, 257]
    check(gpu_device, [(200, 5), (70, 2)], new=new, HQ=HQ, HKV=HKV, D=D, dtype=dtype, before=1, after=1,
          own=lambda n: new[n] + (own if n == 5 else 20 + n))


@pytest.mark.parametrize("N", [2, 64, 65, 255, 256, 300, 1500])
def test_many_groups(N, gpu_device):
    """Plans of one and of several records a thread."""
    check(gpu_device, [(20 + n % 30, 2) for n in range(N // 2)], HQ=2, HKV=1, D=64, after=N % 2, own=lambda n: 1 + n % 7)


def test_more_sequences_than_a_plan_has_room_for(gpu_device):
    check(gpu_device, [(20, 2000), (33, 49)], HQ=1, HKV=1, D=64, own=lambda n: 1 + n % 3)


def test_long_prefixes_are_cut(gpu_device):
    check(gpu_device, [(12000, 2)], HQ=2, HKV=1, D=64)
    check(gpu_device, [(12000, 40)], HQ=2, HKV=1, D=64, own=lambda n: 1 + (n * 41) % 300)
    check(gpu_device, [(5000, 130), (7000, 3)], HQ=4, HKV=1, D=64, own=lambda n: 1 + n % 20)


def test_long_own_tokens_are_cut(gpu_device):
    check(gpu_device, [(100, 3)], HQ=2, HKV=1, own=lambda n: 4000 - 900 * n)
    check(gpu_device, [(1000, 3)], T=40, HQ=2, HKV=1, own=lambda n: 6000 - 900 * n)


def test_ended_and_short_sequences(gpu_device):
    """A freed row, the first of its group, and one whose new tokens begin among
    the shared ones."""
    gen = torch.Generator().manual_seed(7)
    for T in (1, 5):
        kc, vc, table, lens, starts, shared = make([(100, 5), (60, 2)], lambda n: T + 9 * n, 16, 2, 64, BF16, gen)
        lens[0] = 0
        table[0] = -1
        lens[2] = 100 + T - 1  # its first new token is the group's last shared one
        lens[6] = 3  # (with one left, the second group shares nothing)
        q = torch.randn(7, T, 6, 64, generator=gen).to(BF16)
        compare(gpu_device, q, kc, vc, table, lens, starts, shared)
        lens[:] = 0
        compare(gpu_device, q, kc, vc, table, lens, starts, shared)


def test_more_shared_than_there_is(gpu_device):
    """Shared tokens beyond every sequence, or below none."""
    gen = torch.Generator().manual_seed(8)
    kc, vc, table, lens, starts, shared = make([(50, 3), (50, 3)], lambda n: 4, 16, 2, 64, BF16, gen)
    q = torch.randn(6, 2, 4, 64, generator=gen).to(BF16)
    compare(gpu_device, q, kc, vc, table, lens, starts, torch.tensor([1 << 30, -5], dtype=torch.int32))


def test_empty_groups(gpu_device):
    gen = torch.Generator().manual_seed(9)
    kc, vc, table, lens, _, _ = make([(80, 4)], lambda n: 2 + n, 16, 2, 64, BF16, gen)
    q = torch.randn(4, 1, 4, 64, generator=gen).to(BF16)
    for starts, shared in (([0, 0, 4, 4], [7, 80, 9]), ([1, 1, 1, 3], [7, 7, 80]), ([0, 0], [80]), ([4, 4], [80])):
        compare(gpu_device, q, kc, vc, table, lens, *(torch.tensor(x, dtype=torch.int32) for x in (starts, shared)))


def test_offsets_that_are_none_stay_inside(gpu_device):
    """Decreasing offsets, or such outside of the table: results unspecified, no
    access outside of the tensors (the calls after them are right)."""
    gen = torch.Generator().manual_seed(10)
    kc, vc, table, lens, starts, shared = make([(80, 4), (40, 4)], lambda n: 2 + n, 16, 2, 64, BF16, gen)
    q = torch.randn(8, 1, 4, 64, generator=gen).to(BF16)
    args = [t.to(gpu_device) for t in (q, kc, vc, table, lens)]
    for bad in ([0, 8, 0, 8], [5, 3, 1, 0], [-9, 4, 100, 2], [8, 0, 8, 0]):
        paged_attention_shared(*args, torch.tensor(bad, dtype=torch.int32, device=gpu_device),
                               torch.tensor([80, 40, 60], dtype=torch.int32, device=gpu_device))
    cu = torch.tensor([0, 8, 0, 8, 3, 8, 0, 8, 2], dtype=torch.int32, device=gpu_device)
    paged_attention_shared(q.view(1, 8, 4, 64).to(gpu_device), *args[1:], starts.to(gpu_device), shared.to(gpu_device),
                           cu_seqlens=cu)
    torch.cuda.synchronize()
    compare(gpu_device, q, kc, vc, table, lens, starts, shared)
    # a sequence of all 8 tokens several times over: more rows in a group than there are
    kc, vc, table, lens, starts, shared = make([(40, 8)], lambda n: 60 + n, 16, 2, 64, BF16, gen)
    args = [t.to(gpu_device) for t in (q.view(1, 8, 4, 64), kc, vc, table, lens, starts, shared)]
    paged_attention_shared(*args, cu_seqlens=cu)
    torch.cuda.synchronize()
    compare(gpu_device, q, kc, vc, table, lens, starts, shared)


def test_rows_that_there_is_no_room_for_are_nan(gpu_device):
    """256 sequences of all 60 tokens each, by offsets that decrease: their group's
    partial results take 61440 fours of rows, and the room that 60 tokens can need
    is 23020.  No row is left as it was."""
    gen, i32 = torch.Generator().manual_seed(19), dict(dtype=torch.int32, device=gpu_device)
    kc, vc = (torch.randn(64, 16, 16, 64, generator=gen).to(BF16).to(gpu_device) for _ in range(2))
    table = torch.randint(64, (512, 16), generator=gen, dtype=torch.int32).to(gpu_device)
    q = torch.randn(1, 60, 16, 64, generator=gen).to(BF16).to(gpu_device)
    o, lse = paged_attention_shared(q, kc, vc, table, torch.full((512,), 100, **i32), torch.tensor([0, 512], **i32),
                                    torch.tensor([20], **i32), cu_seqlens=torch.tensor([0, 60] * 256 + [0], **i32),
                                    return_lse=True)
    assert bool(o.isnan().all()) and bool(lse.isnan().all())


def test_packed_single_tokens_equal_batch_rows(gpu_device):
    gen = torch.Generator().manual_seed(16)
    kc, vc, table, lens, starts, shared = make([(333, 9), (100, 30)], lambda n: 1 + 9 * n, 16, 4, 128, BF16, gen)
    q = torch.randn(39, 1, 16, 128, generator=gen).to(BF16).to(gpu_device)
    args = [t.to(gpu_device) for t in (kc, vc, table, lens, starts, shared)]
    cu = torch.arange(40, dtype=torch.int32, device=gpu_device)
    want = paged_attention_shared(q, *args, return_lse=True)
    o, lse = paged_attention_shared(q.view(1, 39, 16, 128), *args, cu_seqlens=cu, return_lse=True)
    assert torch.equal(o.view_as(q), want[0]) and torch.equal(lse.view_as(want[1]), want[1])


@pytest.mark.parametrize("T", [1, 8, 40])
def test_one_row_is_read_for_all(T, gpu_device):
    """The other rows' entries for the shared tokens name a page of NaN: what is
    worked on once is read from one row."""
    gen = torch.Generator().manual_seed(11)
    kc, vc, table, lens, starts, shared = make([(160, 4), (64, 9)], lambda n: T + n, 16, 2, 64, BF16, gen)
    q = torch.randn(13, T, 4, 64, generator=gen).to(BF16)
    want = attention(q, kc, vc, table, lens, 64 ** -0.5, lambda pos, j: j <= pos)
    nan = next(p for p in range(kc.shape[0]) if not (table == p).any())
    assert kc[nan].isnan().all() and vc[nan].isnan().all()
    table[1:4, :10] = nan
    table[5:, :4] = nan
    compare(gpu_device, q, kc, vc, table, lens, starts, shared, want=want)


def test_strided_queries(gpu_device):
    gen = torch.Generator().manual_seed(12)
    kc, vc, table, lens, starts, shared = make([(90, 4)], lambda n: 3 + n, 16, 2, 64, BF16, gen)
    qkv = torch.randn(4, 2, 8, 64, generator=gen).to(BF16)
    q = qkv[:, :, 2:6]
    want, want_lse = compare(gpu_device, q.contiguous(), kc, vc, table, lens, starts, shared)
    d = gpu_device
    o, lse = paged_attention_shared(qkv.to(d)[:, :, 2:6], kc.to(d), vc.to(d), table.to(d), lens.to(d), starts.to(d),
                                    shared.to(d), return_lse=True)
    assert torch.equal(o, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("T", [1, 20])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_scores_that_are_not_finite(T, bad, gpu_device):
    """An infinite query makes its own results NaN and no other's."""
    gen = torch.Generator().manual_seed(13)
    kc, vc, table, lens, starts, shared = make([(300, 4)], lambda n: T + 2 + n, 16, 2, 64, BF16, gen)
    d = gpu_device
    q = torch.randn(4, T, 4, 64, generator=gen).to(BF16).to(d)
    args = (kc.to(d), vc.to(d), table.to(d), lens.to(d), starts.to(d), shared.to(d))
    want, want_lse = paged_attention_shared(q, *args, return_lse=True)
    q[2, 0, 1, 0] = bad
    o, lse = paged_attention_shared(q, *args, return_lse=True)
    assert o[2, 0, 1].isnan().all() and lse[2, 0, 1].isnan()
    keep = torch.ones(4, T, 4, dtype=torch.bool, device=d)
    keep[2, 0, 1] = False
    assert torch.equal(o[keep], want[keep]) and torch.equal(lse[keep], want_lse[keep])


def test_answers_forked_from_a_prompt(gpu_device):
    """As it is used: a prompt, forks of it, steps of one token, rows that end;
    every step equals paged_attention's within the rounding of both."""
    d, gen = gpu_device, torch.Generator().manual_seed(14)
    N, page, P, HKV, G, D, L = 6, 16, 60, 2, 4, 64, 150
    pool = torch.randn(2, P, page, HKV, D, generator=gen).to(BF16).to(d)
    i32 = dict(dtype=torch.int32, device=d)
    # (a wide table: the shared keys are worked on together)
    table, lens, refs = torch.full((N, 6000), -1, **i32), torch.zeros(N, **i32), torch.zeros(P, **i32)
    assert bool(paged_reserve(table, lens, refs, torch.tensor([L] + [0] * 5, **i32), page)[0])
    rows = torch.arange(1, N, **i32)
    assert bool(paged_fork(pool, table, lens, refs, torch.zeros_like(rows), rows).all())
    groups, shared = torch.tensor([0, N], **i32), torch.tensor([L], **i32)
    for step in range(20):
        if step == 10:
            paged_free(table, lens, refs, torch.tensor([0, 3], **i32))
        more = (lens > 0).to(torch.int32)
        assert bool(paged_reserve(table, lens, refs, more, page).all())
        x = torch.randn(N, 1, (G + 2) * HKV, D, generator=gen).to(BF16).to(d)
        q, k, v = x.split([G * HKV, HKV, HKV], 2)
        paged_append(k, v, pool[0], pool[1], table, lens)
        o, lse = paged_attention_shared(q, pool[0], pool[1], table, lens, groups, shared, return_lse=True)
        want, want_lse = paged_attention(q, pool[0], pool[1], table, lens, return_lse=True)
        # each rounds its exponentials and its result once: 2^-8 of the weighted |v| (at most 6) and of |o|, twice
        assert (o.float() - want.float()).abs().max().item() <= 2 * 2 * 2.0 ** -8 * 6
        live = lens > 0
        assert (lse - want_lse)[live].abs().max().item() < 1e-4 and (o[~live] == 0).all() and lse[~live].isneginf().all()


def test_another_stream_and_a_graph(gpu_device):
    gen = torch.Generator().manual_seed(15)
    d = gpu_device
    for T, count in ((1, 8), (1, 40), (30, 4)):
        kc, vc, table, lens, starts, shared = make([(700, count), (90, 3)], lambda n: T + 60, 16, 2, 128, BF16, gen)
        kc, vc = kc.nan_to_num().to(d), vc.nan_to_num().to(d)
        table, lens, starts, shared = table.to(d), lens.to(d) - 50, starts.to(d), shared.to(d)
        q = torch.randn(count + 3, T, 8, 128, generator=gen).to(BF16).to(d)

        def step():
            return paged_attention_shared(q, kc, vc, table, lens, starts, shared, return_lse=True)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            there = step()
        torch.cuda.current_stream().wait_stream(side)
        here = step()
        assert torch.equal(here[0], there[0]) and torch.equal(here[1], there[1])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        for i in range(4):
            lens += 7
            if i == 2:
                shared -= 33
            q.copy_(torch.randn(q.shape, generator=gen).to(BF16))
            graph.replay()
            want = step()
            torch.cuda.synchronize()
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype,D,HQ,HKV", [(BF16, 128, 128, 32), (FP16, 64, 128, 32), (BF16, 64, 96, 16)])
@pytest.mark.parametrize("prefix,own", [(200, 20), (9000, 20), (200, 3000)])
def test_sequences_of_many_rows_share_beside_long_chunks(prefix, own, dtype, D, HQ, HKV, gpu_device):
    """Row tiles of 256 (chunks of no group bring their number past three rounds'
    768) beside groups whose records are of many rows too: 12, 20 and 31 new tokens
    (of 6 heads a kv head 21 at most) share with single tokens; the group's keys, or
    a member's own, cut into several parts."""
    G = HQ // HKV
    new = [12, 20, 31 if G == 4 else 21, 1, 9, 20, 500 if HKV == 32 else 900, 257]
    assert all(x * G < 128 for x in new[:6]) and sum(-(-x * G // 128) for x in new) * HKV >= 768
    check(gpu_device, [(prefix, 4), (70, 2)], new=new, HQ=HQ, HKV=HKV, D=D, dtype=dtype, after=2,
          own=lambda n: new[n] + (own if n in (1, 2) else 20 + n))


@pytest.mark.parametrize("D,HQ,HKV,pairs,prefix,own", [
    # tiles of keys times kv heads: 12000 and 24000 (parts of 32 tiles, 64 of head size 64, are finer than a round's),
    # 36000 (1024 parts)
    (128, 32, 32, 4, 3000, 900), (64, 64, 32, 12, 2000, 900), (128, 32, 32, 4, 9000, 60),
    # with no more than 32 rows altogether: waves of fewer, twice the work-groups
    (128, 32, 32, 3, 6000, 700), (64, 32, 16, 8, 9000, 60)])
def test_more_parts_of_few_rows_than_run_at_once(D, HQ, HKV, pairs, prefix, own, gpu_device):
    check(gpu_device, [(prefix + 171 * i, 2) for i in range(pairs)], HQ=HQ, HKV=HKV, D=D, page=64,
          own=lambda n: 1 + (n * 397) % own)
