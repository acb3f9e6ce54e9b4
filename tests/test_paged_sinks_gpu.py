"""Attention with a window and a few first tokens that stay visible, on the GPU
against its definition in 64 bits; bounds as for paged_attention
(tests/paged_bounds.py)."""

from __future__ import annotations

import math

import pytest
import torch

from kda_bt16 import paged_attention
from paged_bounds import misses
from paged_oracle import spans
from paged_seen_oracle import attention, caches, held_tokens, on_device, tables

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def check(dev, lens, window, sinks, T=1, HQ=4, HKV=2, D=128, page=16, dtype=BF16, layout="token", new=None, width=0, seed=0,
          gone="nan"):
    """``gone``: what stands in whole pages of keys that no query sees any more:
    "nan", or the table names no page ("none")."""
    gen = torch.Generator().manual_seed(seed)
    table, P = tables(lens, page, gen, width)
    cu = None if new is None else torch.tensor([0] + new).cumsum(0).to(torch.int32)
    first_seen = [max(0, L - c + 1 - window) for L, (_, c) in zip(lens, spans(len(lens), T, cu))]

    def lost(n, j):  # in a page that lies before the window, behind the first tokens
        return (j // page + 1) * page <= first_seen[n] and j // page * page >= sinks

    kc, vc = caches(table, P, HKV, D, page, dtype, held_tokens(table, P, lens, page, lost), gen, layout)
    if gone == "none":
        for n, L in enumerate(lens):
            for j in range(0, L, page):
                if lost(n, j):
                    table[n, j // page] = -1
    q = torch.randn(*((len(lens), T) if new is None else (1, sum(new))), HQ, D, generator=gen).to(dtype)
    scale = D ** -0.5
    ln = torch.tensor(lens, dtype=torch.int32)
    want = attention(q, kc, vc, table, ln, scale, lambda pos, j: (j > pos - window) | (j < sinks), cu)
    o, lse = paged_attention(q.to(dev), on_device(kc, dev), on_device(vc, dev), table.to(dev), ln.to(dev), scale=scale,
                             window=window, sinks=sinks, cu_seqlens=None if cu is None else cu.to(dev), return_lse=True)
    assert o.shape == q.shape and o.dtype == dtype
    assert not misses(o, lse, want, q, lens, scale, cu)


LENS = [1, 0, 15, 16, 17, 33, 64, 65, 129, 300, 1000]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sinks", [(1, 1), (16, 4), (31, 33), (100, 32), (64, 64), (5, 200), (2000, 3), (100, 5000)])
def test_decode(dtype, D, window, sinks, gpu_device):
    check(gpu_device, LENS, window, sinks, D=D, dtype=dtype)


@pytest.mark.parametrize("gone", ["nan", "none"])
@pytest.mark.parametrize("page", [16, 32, 128, 1024])
@pytest.mark.parametrize("layout", ["token", "head"])
def test_pages_between_are_not_read(gone, page, layout, gpu_device):
    check(gpu_device, [3000, 2048, 1500, 900], 200, 40, page=page, layout=layout, gone=gone)
    check(gpu_device, [3000, 2048, 1500, 900], 200, 40, T=100, page=page, layout=layout, gone=gone)


@pytest.mark.parametrize("T", [2, 5, 31, 64, 100, 129, 300])
@pytest.mark.parametrize("window,sinks", [(1, 1), (50, 4), (64, 70), (333, 64), (7, 129), (128, 1)])
def test_chunks(T, window, sinks, gpu_device):
    check(gpu_device, [T, T + 1, T + 200, T + 63, T + 1100], window, sinks, T=T)


@pytest.mark.parametrize("HQ,HKV", [(1, 1), (3, 1), (10, 2), (32, 1), (40, 1), (16, 16)])
@pytest.mark.parametrize("T", [1, 3, 70])
def test_heads(HQ, HKV, T, gpu_device):
    check(gpu_device, [70, 131, 700], 50, 20, T=T, HQ=HQ, HKV=HKV)


@pytest.mark.parametrize("width", [0, 500])
@pytest.mark.parametrize("D", [64, 128])
def test_packed(width, D, gpu_device):
    check(gpu_device, [5, 0, 900, 64, 1, 1300, 800], 130, 35, new=[5, 0, 200, 1, 1, 1, 513], D=D, width=width)


@pytest.mark.parametrize("N", [1, 8, 70])
def test_work_cut_into_parts(N, gpu_device):
    """Long windows of few rows, and row tiles whose keys go to several work-groups."""
    lens = [6000 - 70 * n for n in range(N)]
    check(gpu_device, lens, 3100, 70, HQ=2, HKV=1)
    if N == 1:
        check(gpu_device, [6000], 4000, 100, T=300, HQ=4, HKV=1)
        check(gpu_device, [6000], 60, 5000, T=300, HQ=4, HKV=1)
        check(gpu_device, [6000], 700, 5900, T=20, HQ=4, HKV=1)
        check(gpu_device, [9000, 5000], 2000, 1000, new=[1, 400], HQ=4, HKV=1)


def test_without_sinks_the_bits_of_the_window(gpu_device):
    """No first tokens, or only such as the window has anyway."""
    gen = torch.Generator().manual_seed(1)
    lens = [500, 90, 300]
    table, P = tables(lens, 16, gen)
    kc, vc = (c.to(gpu_device) for c in caches(table, P, 2, 64, 16, BF16, held_tokens(table, P, lens, 16), gen))
    ln, tb = torch.tensor(lens, dtype=torch.int32, device=gpu_device), table.to(gpu_device)
    for T in (1, 40):
        q = torch.randn(3, T, 8, 64, generator=gen).to(BF16).to(gpu_device)
        want = paged_attention(q, kc, vc, tb, ln, window=100)
        assert torch.equal(paged_attention(q, kc, vc, tb, ln, window=100, sinks=0), want)
        whole = paged_attention(q, kc, vc, tb, ln)
        assert torch.equal(paged_attention(q, kc, vc, tb, ln, window=1000, sinks=7), whole)


def test_a_stream_keeps_its_first_tokens(gpu_device):
    """A first token of high scores holds its weight when the window is far off."""
    gen = torch.Generator().manual_seed(2)
    L, D = 2000, 64
    table, P = tables([L], 16, gen)
    kc, vc = caches(table, P, 1, D, 16, FP16, held_tokens(table, P, [L], 16), gen)
    q = torch.ones(1, 1, 1, D, dtype=FP16)
    first = int(table[0, 0])
    kc[first, 0] = 4.0  # score 4 * 64 / 8 = 32 above the others' (below 12 in 5 standard deviations of 1 each)
    dev = gpu_device
    args = (q.to(dev), kc.to(dev), vc.to(dev), table.to(dev), torch.tensor([L], dtype=torch.int32, device=dev))
    o = paged_attention(*args, window=100, sinks=1)
    # the others' weights: 100 * e^(12 - 32) at most
    assert (o.double().cpu()[0, 0, 0] - vc[first, 0, 0].double()).abs().max().item() <= 12 * 100 * math.exp(-20) + 6 * 2.0 ** -10
    # (without it, the mean of the window's values instead)
    assert (paged_attention(*args, window=100).double().cpu()[0, 0, 0] - vc[first, 0, 0].double()).abs().max().item() > 0.5


def test_another_stream_and_a_graph(gpu_device):
    gen = torch.Generator().manual_seed(3)
    lens = [1500, 40, 900]
    table, P = tables(lens, 16, gen)
    kc, vc = (c.to(gpu_device) for c in caches(table, P, 2, 128, 16, BF16, torch.ones(P, 16, dtype=torch.bool), gen))
    tb, ln = table.to(gpu_device), torch.tensor([1400, 20, 800], dtype=torch.int32, device=gpu_device)
    for T in (1, 50):
        q = torch.randn(3, T, 8, 128, generator=gen).to(BF16).to(gpu_device)

        def step():
            return paged_attention(q, kc, vc, tb, ln, window=900, sinks=33, return_lse=True)

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
        for _ in range(3):
            ln += 5
            q.copy_(torch.randn(q.shape, generator=gen).to(BF16))
            graph.replay()
            want = step()
            torch.cuda.synchronize()
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
