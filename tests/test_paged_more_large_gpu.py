"""First tokens that stay visible, shared first tokens and the append with
rotation on the GPU: caches beyond 2^32 bytes, and random shapes (bounds of
tests/paged_bounds.py)."""

from __future__ import annotations

import random

import pytest
import torch

from kda_bt16 import paged_attention, paged_attention_shared
from paged_bounds import misses
from paged_seen_oracle import attention
from test_paged_rotary_gpu import check as check_rotary
from test_paged_shared_gpu import check as check_shared
from test_paged_sinks_gpu import check as check_sinks

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("T", [1, 40])
def test_caches_past_32_bits(T, gpu_device):
    """Keys and values of 2^32 bytes and more each, the sequences in the last pages."""
    P, page, HKV, D, N = 140, 1024, 128, 128, 3
    gen = torch.Generator().manual_seed(T)
    kc, vc = (torch.zeros(P, page, HKV, D, dtype=BF16, device=gpu_device) for _ in range(2))
    assert kc.numel() * 2 > 1 << 32
    k, v = (torch.randn(N + 1, page, HKV, D, generator=gen).to(BF16) for _ in range(2))
    kc[P - N - 1:], vc[P - N - 1:] = k.to(gpu_device), v.to(gpu_device)
    # two pages a sequence, the first of them shared
    lens = [page + T + 50 * n for n in range(N)]
    small = torch.tensor([[0, 1 + n] for n in range(N)], dtype=torch.int32)
    table = torch.full((N, 64), -1, dtype=torch.int32)  # (room for 256 MB and more of keys and values)
    table[:, :2] = small + P - N - 1
    ln = torch.tensor(lens, dtype=torch.int32)
    q = torch.randn(N, T, HKV, D, generator=gen).to(BF16)
    dev = [t.to(gpu_device) for t in (q,)] + [kc, vc] + [t.to(gpu_device) for t in (table, ln)]
    scale = D ** -0.5
    got = paged_attention_shared(*dev, torch.tensor([0, N], dtype=torch.int32, device=gpu_device),
                                 torch.tensor([page], dtype=torch.int32, device=gpu_device), return_lse=True)
    want = attention(q, k, v, small, ln, scale, lambda pos, j: j <= pos)
    assert not misses(*got, want, q, lens, scale)
    got = paged_attention(*dev, window=300, sinks=70, return_lse=True)
    want = attention(q, k, v, small, ln, scale, lambda pos, j: (j > pos - 300) | (j < 70))
    assert not misses(*got, want, q, lens, scale)


def _shape(rng):
    HKV = rng.choice([1, 1, 2, 3])
    return dict(HKV=HKV, HQ=HKV * rng.choice([1, 2, 3, 5, 8, 17]), D=rng.choice([64, 128]), page=rng.choice([16, 16, 32, 128]),
                dtype=rng.choice([BF16, FP16]), layout=rng.choice(["token", "head"]), seed=rng.randrange(1 << 20))


def _new(rng, N):
    """Tokens of each of N packed sequences, some of none."""
    new = [rng.choice([0, 1, 1, 1, 2, 5, 17, 70]) for _ in range(N)]
    new[rng.randrange(N)] = 3
    return new


@pytest.mark.parametrize("seed", range(40))
def test_random_windows(seed, gpu_device):
    rng = random.Random(seed)
    N, packed = rng.randint(1, 9), rng.random() < 0.5
    new = _new(rng, N) if packed else [rng.choice([1, 1, 2, 4, 30, 90])] * N
    lens = [n + rng.choice([0, 0, 7, 100, 900]) if rng.random() < 0.9 or n else 0 for n in new]
    check_sinks(gpu_device, lens, rng.choice([1, 7, 40, 64, 130, 500]), rng.choice([1, 4, 16, 33, 100, 700]), T=new[0],
                new=new if packed else None, width=rng.choice([0, 0, 200]), gone=rng.choice(["nan", "none"]), **_shape(rng))


@pytest.mark.parametrize("seed", range(60))
def test_random_groups(seed, gpu_device):
    rng = random.Random(1000 + seed)
    groups = [(rng.choice([0, 3, 16, 50, 128, 333, 900]), rng.randint(1, rng.choice([2, 5, 12, 30]))) for _ in
              range(rng.randint(1, 4))]
    before, after = rng.choice([0, 0, 1, 3]), rng.choice([0, 0, 2])
    N, packed = sum(c for _, c in groups) + before + after, rng.random() < 0.5
    new = _new(rng, N) if packed else [rng.choice([1, 1, 2, 4, 20])] * N
    own = [n + rng.choice([0, 0, 5, 40, 300]) for n in new]
    check_shared(gpu_device, groups, own=lambda n: own[n], T=new[0], new=new if packed else None, before=before, after=after,
                 cu_dtype=rng.choice([torch.int32, torch.int64]), **_shape(rng))


@pytest.mark.parametrize("seed", range(40))
def test_random_rotations(seed, gpu_device):
    rng = random.Random(2000 + seed)
    N, packed = rng.choice([1, 2, 5, 70]), rng.random() < 0.5
    new = _new(rng, N) if packed else [rng.choice([1, 1, 2, 9, 40])] * N
    lens = [max(0, n + rng.choice([0, 0, 3, 60, 400, -1])) for n in new]
    kw = _shape(rng)
    check_rotary(gpu_device, lens, T=new[0], new=new if packed else None, extra=rng.choice([0, 3]) if packed else 0,
                 R=rng.choice([16, kw["D"] // 2, kw["D"]]), interleaved=rng.random() < 0.5, inplace=rng.random() < 0.5, **kw)
