"""The append with the position rotation on the GPU against its formula in 64 bits.

Bounds.  A turned pair is off by the angle's error times its size, and the
roundings: the turns, counted in 64 bits, are off by 4e-8 at position 2^30 and
their fraction by 2^-25 once in fp32, together 4.4e-7 in the angle; sine and
cosine in fp32 by 2^-23, the two products' sum by 2^-23: below 2^-20 * (|a| + |b|)
altogether.  Then one rounding to the cache's type: half a step, 2^-8 (bf16) or
2^-11 (fp16) of the value, 2^-25 where fp16 is subnormal.  What is not turned
is moved, and equal.
"""

from __future__ import annotations

import math

import pytest
import torch

from kda_bt16 import paged_append_rotary, paged_attention
from paged_oracle import spans

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
U = {BF16: 2.0 ** -8, FP16: 2.0 ** -11}
TINY = {BF16: 0.0, FP16: 2.0 ** -25}


def turned(x, pos, freq, interleaved):
    """(x turned, how far fp32 may be off) in 64 bits: x [tokens, heads, D]."""
    half = freq.numel()
    angle = pos.double()[:, None, None] * freq.double()
    i = torch.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    x = x.double()
    out, err = x.clone(), torch.zeros_like(x)
    out[..., a] = x[..., a] * angle.cos() - x[..., b] * angle.sin()
    out[..., b] = x[..., b] * angle.cos() + x[..., a] * angle.sin()
    err[..., a] = err[..., b] = 2.0 ** -20 * (x[..., a].abs() + x[..., b].abs())
    return out, err


def within(got, exact, err, dtype, R):
    got, limit = got.double(), err + U[dtype] * (exact.abs() + err) + TINY[dtype]
    assert torch.isfinite(got).all()
    assert bool(((got - exact).abs() <= limit)[..., :R].all()), ((got - exact).abs() / limit)[..., :R].max().item()
    assert torch.equal(got[..., R:], exact[..., R:])


def table_of(lens, page, gen, width=0):
    need = [-(-n // page) for n in lens]
    P = sum(need) + 2
    order = torch.randperm(P, generator=gen, dtype=torch.int32)
    table = torch.full((len(lens), max(need + [1, width])), -1, dtype=torch.int32)
    at = 0
    for n, c in enumerate(need):
        table[n, :c] = order[at:at + c]
        at += c
    return table, P


def check(dev, lens, T=1, HQ=4, HKV=2, D=128, R=None, interleaved=False, page=16, dtype=BF16, layout="token", new=None,
          extra=0, cu_dtype=torch.int32, inplace=False, base=10000.0, hole=None, seed=0):
    """``new``: packed, with ``extra`` tokens behind the last sequence; ``hole``:
    (sequence, entry) of the table that names no page."""
    gen = torch.Generator().manual_seed(seed)
    R = R or D
    table, P = table_of(lens, page, gen)
    if hole:
        table[hole] = -1
    shape = (P, HKV, page, D) if layout == "head" else (P, page, HKV, D)
    caches = [torch.randn(shape, generator=gen).to(dtype).to(dev) for _ in range(2)]
    if layout == "head":
        caches = [c.transpose(1, 2) for c in caches]
    before = [c.cpu().clone() for c in caches]
    cu = None if new is None else torch.tensor([0] + new).cumsum(0).to(cu_dtype)
    N = len(lens)
    lead = (N, T) if new is None else (1, sum(new) + extra)
    qkv = torch.randn(*lead, HQ + 2 * HKV, D, generator=gen).to(dtype)
    freq = (base ** (-torch.arange(R // 2, dtype=torch.float64) / (R // 2))).float()
    here = qkv.to(dev)
    q, k, v = here.split([HQ, HKV, HKV], 2)
    out = paged_append_rotary(q, k, v, *caches, table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), freq.to(dev),
                              interleaved=interleaved, cu_seqlens=None if cu is None else cu.to(dev), out=q if inplace else None)
    assert out.shape == q.shape and out.dtype == dtype
    flat = qkv.reshape(-1, HQ + 2 * HKV, D)
    got = out.cpu().reshape(-1, HQ, D)
    want = [c.double() for c in before]
    err = torch.zeros_like(want[0])
    wrote = torch.zeros(want[0].shape[:2], dtype=torch.bool)
    for n, (first, count) in enumerate(spans(N, T, cu)):
        if count == 0:
            continue
        pos = torch.arange(lens[n] - count, lens[n])
        mine = flat[first:first + count]
        x, e = turned(mine[:, :HQ + HKV], pos, freq, interleaved)
        within(got[first:first + count], x[:, :HQ], e[:, :HQ], dtype, R)
        for i, p in enumerate(pos.tolist()):
            at = int(table[n, p // page]) if p >= 0 else -1
            if at >= 0:
                want[0][at, p % page], err[at, p % page], wrote[at, p % page] = x[i, HQ:], e[i, HQ:], True
                want[1][at, p % page] = mine[i, HQ + HKV:].double()
    k_got, v_got = (c.cpu() for c in caches)
    within(k_got[wrote], want[0][wrote], err[wrote], dtype, R)
    assert torch.equal(k_got[~wrote], before[0][~wrote])
    assert torch.equal(v_got.double(), want[1])
    if extra and inplace:  # tokens of no sequence
        assert torch.equal(here.cpu()[0, -extra:], qkv[0, -extra:])
    assert torch.equal(here.cpu()[:, :, HQ:], qkv[:, :, HQ:])
    if not inplace:
        assert torch.equal(here.cpu(), qkv)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D,R", [(64, 16), (64, 48), (64, 64), (128, 32), (128, 96), (128, 128)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_pairs(dtype, D, R, interleaved, gpu_device):
    check(gpu_device, [1, 0, 17, 500], D=D, R=R, interleaved=interleaved, dtype=dtype)


@pytest.mark.parametrize("T", [1, 2, 7, 64, 301])
@pytest.mark.parametrize("layout", ["token", "head"])
def test_lengths(T, layout, gpu_device):
    # a sequence shorter than its new tokens: those before its first are left out of the cache
    check(gpu_device, [T, T + 15, T + 16, T + 200, T // 2], T=T, layout=layout)


@pytest.mark.parametrize("HQ,HKV", [(1, 1), (3, 1), (5, 2), (32, 8), (24, 4), (70, 2), (2, 8), (64, 64)])
@pytest.mark.parametrize("T", [1, 40])
def test_heads(HQ, HKV, T, gpu_device):
    check(gpu_device, [60, 41, 333], T=T, HQ=HQ, HKV=HKV)


@pytest.mark.parametrize("page", [16, 32, 128, 1024])
@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("cu_dtype", [torch.int32, torch.int64])
def test_packed(page, inplace, cu_dtype, gpu_device):
    check(gpu_device, [5, 0, 900, 64, 1, 130], new=[5, 0, 200, 1, 1, 130], extra=9, page=page, inplace=inplace, cu_dtype=cu_dtype)


@pytest.mark.parametrize("N", [1, 63, 64, 65, 200])
def test_many_sequences(N, gpu_device):
    new = [(7 * n) % 5 for n in range(N)]
    check(gpu_device, [3 + x + n % 40 for n, x in enumerate(new)], new=new[:-1] + [3], HQ=2, HKV=1, D=64)
    check(gpu_device, [4 + n % 40 for n in range(N)], T=2, HQ=2, HKV=1, D=64)


def test_in_place(gpu_device):
    check(gpu_device, [50, 9], T=9, inplace=True)


@pytest.mark.parametrize("shape,order,at", [((9, 5, 8, 64), (1, 0, 2, 3), 2), ((8, 9, 5, 64), (2, 1, 0, 3), 2),
                                            ((5, 9, 2, 3, 64), None, 3), ((9, 5, 2, 3, 64), (1, 0, 2, 3, 4), 3)])
def test_in_place_in_any_order_of_a_projection(shape, order, at, gpu_device):
    """Time first, or every head's query, key and value side by side: the same
    bits as into a new tensor, keys and values left as they were."""
    d, gen = gpu_device, torch.Generator().manual_seed(2)
    buf = torch.randn(shape, generator=gen).to(BF16).to(d)
    x = buf if order is None else buf.permute(order)
    q, k, v = x.split([4, 2, 2], at) if x.ndim == 4 else x.unbind(at)
    lens = [9, 30, 3, 16, 0]
    table, P = table_of(lens, 16, gen)
    table, lens = table.to(d), torch.tensor(lens, dtype=torch.int32, device=d)
    freq = (10000.0 ** (-torch.arange(32) / 32)).to(d)
    there, here = ([torch.zeros(P, 16, 2, 64, dtype=BF16, device=d) for _ in range(2)] for _ in range(2))
    was = [t.clone() for t in (k, v)]
    want = paged_append_rotary(q, k, v, *there, table, lens, freq)
    assert paged_append_rotary(q, k, v, *here, table, lens, freq, out=q) is q
    assert torch.equal(q, want) and all(torch.equal(a, b) for a, b in zip(here + [k, v], there + was))


def test_a_missing_page_is_left_out(gpu_device):
    check(gpu_device, [100, 70], T=60, hole=(0, 4))


@pytest.mark.parametrize("interleaved", [False, True])
def test_far_positions(interleaved, gpu_device):
    """The farthest position that a table can have (2^30 - 1): the angle's turns
    alone fill 24 bits."""
    gen = torch.Generator().manual_seed(3)
    page, M, D, T = 1024, (1 << 20) - 1, 128, 5
    table = torch.full((1, M), -1, dtype=torch.int32)
    table[0, -1] = 1
    L = M * page
    x = torch.randn(1, T, 6, D, generator=gen).to(FP16)
    freq = (500000.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))).float()
    kc, vc = (torch.zeros(2, page, 2, D, dtype=FP16, device=gpu_device) for _ in range(2))
    q, k, v = x.to(gpu_device).split([2, 2, 2], 2)
    out = paged_append_rotary(q, k, v, kc, vc, table.to(gpu_device), torch.tensor([L], dtype=torch.int32, device=gpu_device),
                              freq.to(gpu_device), interleaved=interleaved)
    want, err = turned(x[0, :, :4], torch.arange(L - T, L), freq, interleaved)
    within(out.cpu()[0], want[:, :2], err[:, :2], FP16, D)
    within(kc.cpu()[1, -T:], want[:, 2:], err[:, 2:], FP16, D)
    assert torch.equal(vc.cpu()[1, -T:], x[0, :, 4:]) and not kc.cpu()[0].any() and not kc.cpu()[1, :-T].any()


def test_offsets_past_32_bits(gpu_device):
    """A pool of more than 2^32 bytes of keys, the tokens in its last pages."""
    P, page, HKV, D = 140, 1024, 128, 128
    kc = torch.zeros(P, page, HKV, D, dtype=BF16, device=gpu_device)
    vc = torch.zeros_like(kc)
    assert kc.numel() * 2 > 1 << 32
    table = torch.tensor([[P - 1], [P - 2]], dtype=torch.int32, device=gpu_device)
    lens = torch.tensor([page, 3], dtype=torch.int32, device=gpu_device)
    gen = torch.Generator().manual_seed(4)
    x = torch.randn(2, 2, HKV, D, generator=gen).to(BF16)
    freq = torch.full((D // 2,), 0.01)
    y = x.to(gpu_device)
    paged_append_rotary(y, y, y, kc, vc, table, lens, freq.to(gpu_device))
    for n, L in enumerate((page, 3)):
        want, err = turned(x[n], torch.arange(L - 2, L), freq, False)
        within(kc[P - 1 - n, L - 2:L].cpu(), want, err, BF16, D)
        assert torch.equal(vc[P - 1 - n, L - 2:L].cpu(), x[n])
    assert not kc[:P - 2].any() and not kc[P - 2, 3:].any()


def test_another_stream_and_a_graph(gpu_device):
    """The same bits on a side stream and from a replayed graph, whose replays
    follow the lengths."""
    gen = torch.Generator().manual_seed(5)
    table, P = table_of([100] * 3, 16, gen)
    table = table.to(gpu_device)
    x = torch.randn(3, 1, 8, 64, generator=gen).to(BF16).to(gpu_device)
    freq = torch.rand(32, generator=gen).to(gpu_device)
    q, k, v = x.split([4, 2, 2], 2)
    lens = torch.tensor([7, 50, 99], dtype=torch.int32, device=gpu_device)
    caches = [torch.zeros(P, 16, 2, 64, dtype=BF16, device=gpu_device) for _ in range(4)]

    def step(c):
        return paged_append_rotary(q, k, v, *c, table, lens, freq)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step(caches[2:])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(step(caches[:2]), first) and torch.equal(caches[0], caches[2])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = step(caches[2:])
    for _ in range(3):
        lens += 1
        x.copy_(torch.randn(x.shape, generator=gen).to(BF16))
        graph.replay()
        want = step(caches[:2])
        torch.cuda.synchronize()
        assert torch.equal(o, want)
        assert torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])


def test_scores_depend_on_distances_alone(gpu_device):
    """Used as it is meant: two sequences with the same tokens, the second's all
    1000 positions on (behind keys far below the others' scores), attend alike."""
    gen = torch.Generator().manual_seed(6)
    D, T, far = 64, 40, 1000
    table, P = table_of([T, T + far], 16, gen)
    kc, vc = (torch.zeros(P, 16, 1, D, dtype=FP16, device=gpu_device) for _ in range(2))
    x = torch.randn(1, T, 4, D, generator=gen).to(FP16)
    x = torch.cat([x, x]).to(gpu_device)
    freq = (10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))).float().to(gpu_device)
    lens = torch.tensor([T, T + far], dtype=torch.int32, device=gpu_device)
    q, k, v = x.split([2, 1, 1], 2)
    q = paged_append_rotary(q, k, v, kc, vc, table.to(gpu_device), lens, freq)
    o = paged_attention(q, kc, vc, table.to(gpu_device), lens, window=T, scale=0.1).float().cpu()
    # (of the second's queries the last sees its own T tokens alone)
    # scores are sums of 64 products of turned queries and keys, each off by 2^-11 of its size twice: their sum by
    # 2 * 2^-11 * 0.1 * 64 at most (unit variance), the weights by that, o by twice it of |v| < 4 and its own roundings
    assert (o[0, -1] - o[1, -1]).abs().max().item() < 2 * 2 * 2.0 ** -11 * 0.1 * 64 * 4 + 4 * 2.0 ** -10
    assert math.isfinite(o.sum().item())
