"""The paged cache on the GPU against its plain form in 64 bits.

Attention's tolerances.  With unit-variance q, k, v and scale D^-0.5 the
outputs are weighted means of v.  Each weight e^(s-m) is rounded once to the
cache's type (relative error at most u, 2^-9 for bf16, 2^-12 for fp16) and o
once more; sums are fp32.  So |o - exact| <= u * sum(w |v|) + u |o| plus fp32
rounding of the scores (D products of size ~1: below 1e-4 absolute for the
sizes here): at most 2 * u * max|v| + 1e-4, with max|v| <= 6.  The log-sum-exp
is fp32 throughout: 1e-4 absolute (scores) is ample.
"""

from __future__ import annotations

import math

import pytest
import torch

import paged_oracle as oracle
from kda_bt16 import (
    paged_append,
    paged_attention,
    paged_compact,
    paged_copy,
    paged_fork,
    paged_free,
    paged_reserve,
)

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -12}
BF16, FP16 = torch.bfloat16, torch.float16


def _tol(dtype):
    return 2 * U[dtype] * 6 + 1e-4


def make(lens, HKV, D, page, dtype, dev, layout="token", seed=0, spare=2, width=0):
    """A cache whose unused places hold NaN, its table (with unused entries
    -1) and lengths."""
    gen = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    P = sum(need) + spare
    order = torch.randperm(P, generator=gen, dtype=torch.int32)
    M = max(max(need), width, 1)
    table = torch.full((len(lens), M), -1, dtype=torch.int32)
    at = 0
    caches = []
    for n, c in enumerate(need):
        table[n, :c] = order[at:at + c]
        at += c
    for _ in range(2):
        shape = (P, HKV, page, D) if layout == "head" else (P, page, HKV, D)
        c = torch.randn(shape, generator=gen).clamp(-6, 6).to(dtype)
        c = c.transpose(1, 2) if layout == "head" else c
        held = torch.zeros(P, page, dtype=torch.bool)
        for n, L in enumerate(lens):
            for j in range(need[n]):
                held[int(table[n, j]), :min(page, L - j * page)] = True
        c[~held] = math.nan
        caches.append(c)
    dc = [(c.transpose(1, 2).contiguous().to(dev).transpose(1, 2) if layout == "head" else c.to(dev)) for c in caches]
    ln = torch.tensor(lens, dtype=torch.int32)
    return caches, dc, table, ln, gen


def check(lens, T, HQ, HKV, D, page, dtype, dev, layout="token", causal=True, window=None, new=None, seed=0, scale=None,
          cu_dtype=torch.int32):
    (kc, vc), (dk, dv), table, ln, gen = make(lens, HKV, D, page, dtype, dev, layout, seed)
    N = len(lens)
    cu = None
    if new is not None:
        cu = torch.tensor([0] + new).cumsum(0).to(cu_dtype)
        shape = (1, sum(new), HQ, D)
    else:
        shape = (N, T, HQ, D)
    q = torch.randn(shape, generator=gen).to(dtype)
    scale = D ** -0.5 if scale is None else scale
    want, want_lse = oracle.attention(q, kc, vc, table, ln, scale, causal, window, cu)
    o, lse = paged_attention(q.to(dev), dk, dv, table.to(dev), ln.to(dev), scale=scale, causal=causal, window=window,
                             cu_seqlens=None if cu is None else cu.to(dev), return_lse=True)
    assert o.shape == q.shape and o.dtype == dtype and lse.dtype == torch.float32
    o, lse = o.double().cpu(), lse.double().cpu()
    none = torch.isneginf(want_lse)
    assert torch.equal(torch.isneginf(lse), none)
    assert (o[none] == 0).all()
    assert torch.isfinite(o).all()
    err = (o - want).abs().max().item()
    assert err <= _tol(dtype), f"o off by {err}"
    if (~none).any():
        err = (lse - want_lse)[~none].abs().max().item()
        assert err <= 1e-4, f"lse off by {err}"


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("layout", ["token", "head"])
def test_decode_lengths(dtype, D, layout, gpu_device):
    # around the tile and page borders, one key, none
    lens = [1, 0, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 257]
    check(lens, 1, 8, 2, D, 16, dtype, gpu_device, layout)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 1024])
def test_page_sizes(page, gpu_device):
    check([1, 100, 1025, 700], 3, 4, 2, 128, page, BF16, gpu_device)


@pytest.mark.parametrize("HQ,HKV", [(1, 1), (2, 2), (3, 1), (12, 2), (10, 2), (32, 1), (40, 1), (16, 16), (70, 2)])
@pytest.mark.parametrize("T", [1, 3])
def test_head_groups(HQ, HKV, T, gpu_device):
    check([5, 131, 64], T, HQ, HKV, 128, 16, BF16, gpu_device)


@pytest.mark.parametrize("T", [2, 5, 31, 32, 33, 64, 100, 129, 300])
@pytest.mark.parametrize("D", [64, 128])
def test_chunk_lengths(T, D, gpu_device):
    check([T, T + 1, T + 200, T + 63], T, 4, 2, D, 16, BF16, gpu_device)


@pytest.mark.parametrize("T", [4, 150])
def test_rows_that_see_nothing(T, gpu_device):
    # fewer cached tokens than new ones: the first queries sit before the start
    check([0, 1, 2, T - 1, T], T, 4, 2, 128, 16, BF16, gpu_device)


@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 100, 1000])
@pytest.mark.parametrize("T", [1, 7, 140])
def test_window(window, T, gpu_device):
    check([T, T + 65, 333 + T, 640], T, 4, 2, 128, 16, BF16, gpu_device, window=window)


@pytest.mark.parametrize("T", [1, 6, 130])
def test_not_causal(T, gpu_device):
    check([3, 0, 64, 400], T, 6, 2, 64, 32, FP16, gpu_device, causal=False)


@pytest.mark.parametrize("cu_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("window", [None, 50])
def test_packed(cu_dtype, window, gpu_device):
    new = [1, 0, 40, 1, 129, 0, 3, 17]
    lens = [300, 20, 40, 1, 150, 0, 2, 500]
    check(lens, 0, 8, 2, 128, 16, BF16, gpu_device, new=new, cu_dtype=cu_dtype, window=window)


def test_packed_many_sequences(gpu_device):
    gen = torch.Generator().manual_seed(5)
    new = torch.randint(0, 4, (150,), generator=gen).tolist()
    lens = [n + int(x) for n, x in zip(new, torch.randint(0, 90, (150,), generator=gen))]
    check(lens, 0, 4, 1, 64, 16, BF16, gpu_device, new=new)


@pytest.mark.parametrize("T", [1, 40])
def test_long_context(T, gpu_device):
    check([5000, 3001], T, 4, 2, 128, 32, BF16, gpu_device)


@pytest.mark.parametrize("causal, window", [(True, None), (True, 4200), (False, None)])
@pytest.mark.parametrize("D", [64, 128])
def test_long_contexts_taken_whole(D, causal, window, gpu_device):
    """More row tiles than half the work-groups that run at once: each goes
    over all of its keys, more than 64 tiles of them, in one piece."""
    lens = [9000, 4099, 8192] + [5 + 3 * n % 60 for n in range(130)]
    check(lens, 5, 8, 1, D, 16, BF16, gpu_device, causal=causal, window=window)


@pytest.mark.parametrize("T", [1, 16, 140])
def test_large_scores(T, gpu_device):
    """Scores of some hundreds: the running maximum moves far, most weights
    vanish.  The bound on o holds as it is (weights sum to 1); a score of size
    400 in fp32 is off by 400 * 2^-24 * sqrt(D), far below 1e-3, which moves
    the weights by as much."""
    (kc, vc), (dk, dv), table, ln, gen = make([70, 1200], 2, 128, 16, BF16, gpu_device)
    q = (8 * torch.randn(2, T, 8, 128, generator=gen)).to(BF16)
    want, want_lse = oracle.attention(q, kc, vc, table, ln, 1.0)
    o, lse = paged_attention(q.to(gpu_device), dk, dv, table.to(gpu_device), ln.to(gpu_device), scale=1.0,
                             return_lse=True)
    assert (o.double().cpu() - want).abs().max() <= _tol(BF16) + 6e-3
    assert torch.equal(torch.isneginf(lse.cpu()), torch.isneginf(want_lse))
    some = ~torch.isneginf(want_lse)
    assert (lse.double().cpu() - want_lse)[some].abs().max() <= 2e-3


def test_strided_queries_and_rows(gpu_device):
    """q a slice of a fused projection, the table a slice of a wider one, the
    cache a layer of a larger tensor."""
    dev = gpu_device
    lens, page, HKV, D = [90, 33], 16, 2, 128
    (kc, vc), _, table, ln, gen = make(lens, HKV, D, page, BF16, dev)
    both = torch.stack([kc, vc]).to(dev)  # [2, P, page, HKV, D]
    wide = torch.full((2, table.shape[1] + 5), 7, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    qkv = torch.randn(2, 3, 8 + 4, D, generator=gen).to(BF16)
    want, _ = oracle.attention(qkv[:, :, 2:10], kc, vc, table, ln, 0.1)
    o = paged_attention(qkv.to(dev)[:, :, 2:10], both[0], both[1], wide.to(dev)[:, :table.shape[1]], ln.to(dev),
                        scale=0.1)
    assert (o.double().cpu() - want).abs().max() <= _tol(BF16)


@pytest.mark.parametrize("T", [1, 5, 150])
def test_pages_before_the_window_may_be_gone(T, gpu_device):
    """A window's cache lets pages go once every query is past them: their
    entries may be -1, or pages that hold anything by now."""
    dev, page, window = gpu_device, 16, 70
    lens = [T + 90, T + 333, T + 1000, T + 16]
    (kc, vc), _, table, ln, gen = make(lens, 2, 128, page, BF16, dev)
    q = torch.randn(4, T, 8, 128, generator=gen).to(BF16)
    want, want_lse = oracle.attention(q, kc, vc, table, ln, 0.1, window=window)
    for n, L in enumerate(lens):
        gone = max(0, L - T + 1 - window) // page
        for j in range(gone):
            kc[int(table[n, j])], vc[int(table[n, j])] = math.nan, math.inf
            if j % 2:
                table[n, j] = -1
    o, lse = paged_attention(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev), ln.to(dev), scale=0.1, window=window,
                             return_lse=True)
    assert (o.double().cpu() - want).abs().max() <= _tol(BF16)
    assert (lse.double().cpu() - want_lse).abs().max() <= 1e-4


def test_attention_repeats_its_bits(gpu_device):
    dev = gpu_device
    _, (dk, dv), table, ln, gen = make([3000, 17, 901], 2, 128, 16, BF16, dev)
    q = torch.randn(3, 4, 8, 128, generator=gen).to(BF16).to(dev)
    a = [paged_attention(q, dk, dv, table.to(dev), ln.to(dev), return_lse=True) for _ in range(3)]
    for o, lse in a[1:]:
        assert torch.equal(o, a[0][0]) and torch.equal(lse, a[0][1])


def test_malformed_tables_stay_inside(gpu_device):
    """Entries and lengths outside their ranges: any result, no access
    outside the tensors (the kernels clamp them), and the other sequences'
    results as ever."""
    dev = gpu_device
    (kc, vc), (dk, dv), table, ln, gen = make([100, 80, 60], 2, 128, 16, BF16, dev)
    q = torch.randn(3, 2, 4, 128, generator=gen).to(BF16)
    want, _ = oracle.attention(q, kc, vc, table, ln, 0.1)
    bad, bl = table.clone(), ln.clone()
    bad[0, 1], bad[0, 3] = -7, 1 << 30
    bl[1] = 1 << 30
    o = paged_attention(q.to(dev), dk, dv, bad.to(dev), bl.to(dev), scale=0.1)
    assert (o[2].double().cpu() - want[2]).abs().max() <= _tol(BF16)


# -- append ---------------------------------------------------------------


@pytest.mark.parametrize("dtype,D,layout,HKV", [(BF16, 128, "token", 2), (FP16, 64, "head", 3), (BF16, 64, "token", 1)])
@pytest.mark.parametrize("packed", [False, True])
def test_append(dtype, D, layout, HKV, packed, gpu_device):
    dev = gpu_device
    lens = [40, 17, 16, 3, 0, 130]
    new = [5, 1, 16, 7, 2, 33] if packed else None
    (kc, vc), (dk, dv), table, ln, gen = make(lens, HKV, D, 16, dtype, dev, layout)
    table[0, 1] = -1  # a page that is missing
    cu = torch.tensor([0] + new).cumsum(0) if packed else None
    shape = (1, sum(new)) if packed else (6, 20)
    kv = torch.randn(*shape, 2 * HKV, D, generator=gen).to(dtype)
    k, v = kv[:, :, :HKV], kv[:, :, HKV:]
    oracle.append(k, v, kc, vc, table, ln, cu)
    dkv = kv.to(dev)
    paged_append(dkv[:, :, :HKV], dkv[:, :, HKV:], dk, dv, table.to(dev), ln.to(dev),
                 cu_seqlens=None if cu is None else cu.to(dev))
    for want, got in ((kc, dk), (vc, dv)):
        assert torch.equal(want.contiguous().view(torch.int16), got.cpu().contiguous().view(torch.int16))


# -- pages ----------------------------------------------------------------


class Pages:
    """Random tables on both sides: lists for the oracle, tensors for the GPU."""

    def __init__(self, N, M, P, size, dev, seed, lead=(3,), page=(4, 8), dtype=torch.float32, used=0.6):
        gen = torch.Generator().manual_seed(seed)
        self.size, self.dev = size, dev
        self.refs, self.lens = [0] * P, [0] * N
        self.table = [[-1] * M for _ in range(N)]
        order, at = torch.randperm(P, generator=gen).tolist(), 0
        for n in range(N):
            pages = int(torch.randint(0, M + 1, (1,), generator=gen))
            if at + pages > used * P:
                break
            for j in range(pages):
                self.table[n][j] = order[at]
                self.refs[order[at]] = 1
                at += 1
            tail = int(torch.randint(0, size, (1,), generator=gen)) if pages else 0
            self.lens[n] = pages * size - tail
        self.pool = torch.randn(*lead, P, size, *page, generator=gen).to(dtype)
        self.d_pool = self.pool.to(dev)
        self.d_refs, self.d_lens, self.d_table = self.ints(self.refs), self.ints(self.lens), self.ints(self.table)

    def ints(self, x):
        return torch.tensor(x, dtype=torch.int32, device=self.dev)

    def flat(self):
        return self.pool.view(-1, *self.pool.shape[-4:])

    def same(self, pool=True):
        assert self.d_table.tolist() == self.table
        assert self.d_lens.tolist() == self.lens
        assert self.d_refs.tolist() == self.refs
        if pool:
            assert torch.equal(self.d_pool.cpu(), self.pool)


@pytest.mark.parametrize("N,M,P,size", [(1, 1, 1, 16), (5, 7, 40, 16), (70, 9, 700, 32), (3, 300, 5000, 16),
                                        (1500, 4, 9001, 16)])
def test_reserve_and_free(N, M, P, size, gpu_device):
    s = Pages(N, M, P, size, gpu_device, N + P)
    gen = torch.Generator().manual_seed(N)
    for step in range(3):
        more = torch.randint(-1, 3 * size, (N,), generator=gen).tolist()
        ok = paged_reserve(s.d_table, s.d_lens, s.d_refs, s.ints(more), size)
        assert ok.tolist() == oracle.reserve(s.table, s.lens, s.refs, more, size)
        s.same()
        rows = torch.randperm(N, generator=gen)[:max(1, N // 3)].tolist()
        paged_free(s.d_table, s.d_lens, s.d_refs, s.ints(rows))
        oracle.free(s.table, s.lens, s.refs, rows)
        s.same()


def test_reserve_runs_out(gpu_device):
    s = Pages(4, 8, 6, 16, gpu_device, 1, used=0)
    more = [33, 200, 40, 1]  # 3 pages; more than a row holds; 3 pages; one that is not there
    ok = paged_reserve(s.d_table, s.d_lens, s.d_refs, s.ints(more), 16)
    assert ok.tolist() == oracle.reserve(s.table, s.lens, s.refs, more, 16) == [True, False, True, False]
    s.same()


def test_free_twice_and_rows_outside(gpu_device):
    s = Pages(5, 6, 40, 16, gpu_device, 3)
    paged_free(s.d_table, s.d_lens, s.d_refs, s.ints([1, 1, -1, 99, 1]))
    oracle.free(s.table, s.lens, s.refs, [1])
    s.same()
    paged_free(s.d_table, s.d_lens, s.d_refs, s.ints([]))
    s.same()


@pytest.mark.parametrize("N,M,P,size", [(4, 5, 30, 16), (40, 20, 900, 16), (600, 3, 4100, 32)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_fork(N, M, P, size, dtype, gpu_device):
    s = Pages(N, M, P, size, gpu_device, N, dtype=dtype)
    gen = torch.Generator().manual_seed(N)
    rows = torch.randperm(N, generator=gen).tolist()
    dst, keep = rows[:N // 2], rows[N // 2:]
    src = [keep[int(i)] for i in torch.randint(0, len(keep), (len(dst),), generator=gen)]
    paged_free(s.d_table, s.d_lens, s.d_refs, s.ints(dst))
    oracle.free(s.table, s.lens, s.refs, dst)
    ok = paged_fork(s.d_pool, s.d_table, s.d_lens, s.d_refs, s.ints(src), s.ints(dst))
    assert ok.tolist() == oracle.fork([s.flat()], s.table, s.lens, s.refs, src, dst, size)
    s.same()


def test_fork_runs_out(gpu_device):
    s = Pages(6, 2, 4, 16, gpu_device, 0, used=0)
    s.table[0], s.refs[2], s.lens[0] = [2, -1], 1, 5
    s.d_refs, s.d_lens, s.d_table = s.ints(s.refs), s.ints(s.lens), s.ints(s.table)
    src, dst = [0] * 5, [1, 2, 3, 4, 5]
    ok = paged_fork(s.d_pool, s.d_table, s.d_lens, s.d_refs, s.ints(src), s.ints(dst))
    assert ok.tolist() == oracle.fork([s.flat()], s.table, s.lens, s.refs, src, dst, 16)
    assert ok.tolist() == [True, True, True, False, False]
    s.same()


@pytest.mark.parametrize("N,M,P,used", [(4, 5, 30, 0.6), (40, 20, 900, 0.9), (700, 12, 9500, 0.5), (2, 3, 7, 0.0),
                                        (8, 16, 64, 1.0), (3, 2, 4096, 0.5), (3, 2, 4097, 0.5)])
def test_compact(N, M, P, used, gpu_device):
    s = Pages(N, M, P, 16, gpu_device, P, lead=(2, 2), used=used)
    before = s.d_table.clone(), s.d_refs.clone()
    table, refs, live = paged_compact(s.d_pool, s.d_table, s.d_refs)
    w_table, w_refs, w_live = oracle.compact([s.flat()], s.table, s.refs)
    assert live.tolist() == [w_live]
    assert table.tolist() == w_table and refs.tolist() == w_refs
    assert torch.equal(s.d_pool.cpu(), s.pool)
    assert torch.equal(before[0], s.d_table) and torch.equal(before[1], s.d_refs)


def test_copy_of_several_pools_of_any_type(gpu_device):
    gen = torch.Generator().manual_seed(0)
    # pages of 32 bytes, of 48 KiB + 16, recurrent states
    pools = [torch.randn(5, 9, 2, 2, 4, generator=gen).to(BF16), torch.randn(9, 1, 3, 4097 * 4, generator=gen).contiguous(),
             torch.randn(2, 3, 9, 2, 128, 128, generator=gen)]
    got = [t.to(gpu_device) for t in pools]
    src, dst = [0, 8, -1, 4, 4, 3], [1, 2, 3, 9, 5, 7]
    paged_copy(got, *(torch.tensor(x, dtype=torch.int32, device=gpu_device) for x in (src, dst)))
    for t in pools:
        for a, b in ((0, 1), (8, 2), (4, 5), (3, 7)):
            t[..., b, :, :, :] = t[..., a, :, :, :].clone()
    for want, out in zip(pools, got):
        assert torch.equal(out.cpu(), want)


def test_other_stream_than_the_tensors_own(gpu_device):
    dev = gpu_device
    (kc, vc), (dk, dv), table, ln, gen = make([300, 77], 2, 128, 16, BF16, dev)
    q = torch.randn(2, 2, 8, 128, generator=gen).to(BF16)
    want, _ = oracle.attention(q, kc, vc, table, ln, 0.1)
    args = q.to(dev), dk, dv, table.to(dev), ln.to(dev)
    side = torch.cuda.Stream(device=dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        o = paged_attention(*args, scale=0.1)
    torch.cuda.current_stream(dev).wait_stream(side)
    assert (o.double().cpu() - want).abs().max() <= _tol(BF16)
