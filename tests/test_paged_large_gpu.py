"""Paged calls over pools whose offsets pass 32 bits, many sequences, and
random shapes."""

from __future__ import annotations

import random

import pytest
import torch

import paged_oracle as oracle
from kda_bt16 import paged_append, paged_attention, paged_compact, paged_copy
from test_paged_gpu import BF16, FP16, _tol, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 50])
@pytest.mark.parametrize("layout", ["pages", "heads"])
def test_offsets_past_32_bits(T, layout, gpu_device):
    """A cache of 4.6 GB each for keys and values whose last pages are used:
    element offsets above 2^31, byte offsets above 2^32.  "heads": the heads
    outermost, so that the head's stride passes them."""
    dev, page, HKV, D = gpu_device, 16, 8, 128
    P = 140_000
    shape = (P, page, HKV, D) if layout == "pages" else (HKV, P, page, D)
    kc, vc = (torch.empty(shape, dtype=BF16, device=dev) for _ in range(2))
    if layout == "heads":
        kc, vc = (t.permute(1, 2, 0, 3) for t in (kc, vc))
    lens = torch.tensor([100, 64], dtype=torch.int32)
    table = torch.tensor([[P - 1, 3, P - 2, P - 5, 0, 1, P - 7], [P - 3, 7, P - 4, P - 6, -1, -1, -1]], dtype=torch.int32)
    gen = torch.Generator().manual_seed(1)
    small_k = torch.randn(11, page, HKV, D, generator=gen).to(BF16)
    small_v = torch.randn(11, page, HKV, D, generator=gen).to(BF16)
    small_table = torch.tensor([[0, 1, 2, 3, 4, 5, 6], [7, 8, 9, 10, -1, -1, -1]], dtype=torch.int32)
    at = table.flatten()[table.flatten() >= 0].long().to(dev)
    kc[at], vc[at] = small_k.to(dev), small_v.to(dev)
    new_k, new_v = (torch.randn(2, T, HKV, D, generator=gen).to(BF16) for _ in range(2))
    paged_append(new_k.to(dev), new_v.to(dev), kc, vc, table.to(dev), lens.to(dev))
    oracle.append(new_k, new_v, small_k, small_v, small_table, lens)
    assert torch.equal(kc[at].cpu(), small_k) and torch.equal(vc[at].cpu(), small_v)
    q = torch.randn(2, T, 8, D, generator=gen).to(BF16)
    want, _ = oracle.attention(q, small_k, small_v, small_table, lens, 0.1)
    o = paged_attention(q.to(dev), kc, vc, table.to(dev), lens.to(dev), scale=0.1)
    assert (o.double().cpu() - want).abs().max() <= _tol(BF16)


def test_pages_of_a_pool_past_32_bits(gpu_device):
    """A pool of 2 x 140,000 pages of 32 KB, 9.2 GB."""
    dev, P = gpu_device, 140_000
    pool = torch.empty(2, P, 16, 8, 128, dtype=BF16, device=dev)
    gen = torch.Generator(device=dev).manual_seed(0)
    src = torch.tensor([P - 1, P - 3, 5], dtype=torch.int32, device=dev)
    dst = torch.tensor([2, P - 8, P - 2], dtype=torch.int32, device=dev)
    data = torch.randn(2, 3, 16, 8, 128, generator=gen, device=dev).to(BF16)
    pool[:, src.long()] = data
    paged_copy(pool, src, dst)
    assert torch.equal(pool[:, dst.long()], data)
    # all but the pages of dst are free: they move to the first three places
    refs = torch.zeros(P, dtype=torch.int32, device=dev)
    refs[dst.long()] = torch.tensor([1, 2, 3], dtype=torch.int32, device=dev)
    table = torch.tensor([[2, P - 8], [P - 2, -1]], dtype=torch.int32, device=dev)
    new, new_refs, live = paged_compact(pool, table, refs)
    assert live.tolist() == [3]
    assert new.tolist() == [[2, 0], [1, -1]]
    assert new_refs[:4].tolist() == [2, 3, 1, 0] and int(new_refs.sum()) == 6
    assert torch.equal(pool[:, torch.tensor([2, 0, 1], device=dev)], data)


@pytest.mark.parametrize("T", [1, 2])
def test_thousands_of_sequences(T, gpu_device):
    gen = torch.Generator().manual_seed(T)
    lens = torch.randint(0, 60, (3000,), generator=gen).tolist()
    check(lens, T, 2, 1, 64, 16, BF16, gpu_device)


@pytest.mark.parametrize("seed", range(40))
def test_random_shapes(seed, gpu_device):
    rng = random.Random(seed)
    HKV = rng.choice([1, 2, 3])
    HQ = HKV * rng.choice([1, 2, 3, 5, 8])
    N = rng.choice([1, 2, 5, 9])
    T = rng.choice([1, 1, 2, 7, 33, 90, 270])
    T = max(1, min(T, 900 // N))
    lens = [rng.choice([0, rng.randint(1, 40), rng.randint(1, 700), rng.randint(1, 1800)]) for _ in range(N)]
    new = [rng.choice([0, 1, rng.randint(1, T)]) for _ in range(N)] if rng.random() < 0.5 else None
    if new and sum(new) == 0:
        new[0] = 1
    causal = rng.random() < 0.8
    window = rng.choice([None, None, rng.randint(1, 300)]) if causal else None
    check(lens, T, HQ, HKV, rng.choice([64, 128]), rng.choice([16, 32, 128]), rng.choice([BF16, FP16]), gpu_device,
          rng.choice(["token", "head"]), causal, window, new, seed, cu_dtype=rng.choice([torch.int32, torch.int64]))
