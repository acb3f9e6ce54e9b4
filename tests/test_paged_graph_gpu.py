"""Paged calls in a captured graph: replays between eager work give the eager
results, for lengths and tables that change in place."""

from __future__ import annotations

import pytest
import torch

from kda_bt16 import paged_append, paged_attention, paged_reserve

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 40])
def test_a_captured_step_replays(T, gpu_device):
    dev, page, HQ, HKV, D, N = gpu_device, 16, 8, 2, 128, 3
    gen = torch.Generator(device=dev).manual_seed(T)
    P, M = 200, 60
    kc = torch.randn(P, page, HKV, D, generator=gen, device=dev).bfloat16()
    vc = torch.randn(P, page, HKV, D, generator=gen, device=dev).bfloat16()
    table = torch.full((N, M), -1, dtype=torch.int32, device=dev)
    lens = torch.zeros(N, dtype=torch.int32, device=dev)
    refs = torch.zeros(P, dtype=torch.int32, device=dev)
    start = torch.tensor([5, 400, 130], dtype=torch.int32, device=dev)
    assert paged_reserve(table, lens, refs, start, page).all()
    more = torch.full((N,), T, dtype=torch.int32, device=dev)
    q = torch.empty(N, T, HQ, D, dtype=torch.bfloat16, device=dev)
    k = torch.empty(N, T, HKV, D, dtype=torch.bfloat16, device=dev)
    v = torch.empty_like(k)

    def step(table, lens, refs, kc, vc):
        ok = paged_reserve(table, lens, refs, more, page)
        paged_append(k, v, kc, vc, table, lens)
        return ok, *paged_attention(q, kc, vc, table, lens, return_lse=True)

    eager = [t.clone() for t in (table, lens, refs, kc, vc)]
    step(*[t.clone() for t in eager])  # warm up outside the capture
    held = [table, lens, refs, kc, vc]
    side = torch.cuda.Stream(device=dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step(*held)
    for _ in range(4):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=gen, device=dev))
        graph.replay()
        torch.cuda.synchronize(dev)
        want = step(*eager)
        for a, b in zip(out, want):
            assert torch.equal(a, b)
        for a, b in zip(held, eager):
            assert torch.equal(a, b)
