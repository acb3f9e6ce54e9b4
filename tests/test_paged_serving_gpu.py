"""The paged cache's calls together, as a serving loop makes them, on the GPU:
prompts appended with their rotation and attended to, answers forked from them
that share the prompt, rows that end, the pool compacted, and a window with
first tokens over what has grown.

After every call what the caches hold is checked against the formula in 64 bits
(the bounds of test_paged_rotary_gpu.py), and attention against the caches
(paged_bounds.py)."""

from __future__ import annotations

import pytest
import torch

from kda_bt16 import (
    paged_append,
    paged_append_rotary,
    paged_attention,
    paged_attention_shared,
    paged_compact,
    paged_fork,
    paged_free,
    paged_reserve,
)
from paged_bounds import misses
from paged_seen_oracle import attention
from test_paged_rotary_gpu import turned, within

pytestmark = pytest.mark.gpu

PAGE, HQ, HKV, D, R = 16, 8, 2, 64, 32


class Loop:
    """Rows of a cache, what was appended to each of them (on the CPU, before its
    rotation), and the calls with their checks."""

    def __init__(self, dev, rows, pages, width, dtype, seed):
        self.dev, self.dtype, self.gen = dev, dtype, torch.Generator().manual_seed(seed)
        i32 = dict(dtype=torch.int32, device=dev)
        self.pool = torch.zeros(2, pages, PAGE, HKV, D, dtype=dtype, device=dev)
        self.table, self.lens = torch.full((rows, width), -1, **i32), torch.zeros(rows, **i32)
        self.refs = torch.zeros(pages, **i32)
        self.freq = (10000.0 ** (-torch.arange(R // 2, dtype=torch.float64) / (R // 2))).float()
        self.keys = [torch.zeros(0, HKV, D, dtype=dtype) for _ in range(rows)]
        self.values = [torch.zeros(0, HKV, D, dtype=dtype) for _ in range(rows)]

    def i32(self, x):
        return torch.tensor(x, dtype=torch.int32, device=self.dev)

    def append(self, new, cu=None):
        """New tokens of every row: ``new[n]`` of them.  The turned queries."""
        assert bool(paged_reserve(self.table, self.lens, self.refs, self.i32(new), PAGE).all())
        shape = (1, sum(new)) if cu is not None else (len(new), max(new))
        qkv = torch.randn(*shape, HQ + 2 * HKV, D, generator=self.gen).to(self.dtype)
        flat, at = qkv.reshape(-1, HQ + 2 * HKV, D), 0
        for n, count in enumerate(new):
            width = count if cu is not None else max(new)
            mine = flat[at:at + width]
            at += width
            if count:
                self.keys[n] = torch.cat([self.keys[n], mine[:, HQ:HQ + HKV]])
                self.values[n] = torch.cat([self.values[n], mine[:, HQ + HKV:]])
        q, k, v = qkv.to(self.dev).split([HQ, HKV, HKV], 2)
        q = paged_append_rotary(q, k, v, self.pool[0], self.pool[1], self.table, self.lens, self.freq.to(self.dev),
                                cu_seqlens=cu)
        kc, vc, table = self.pool[0].cpu(), self.pool[1].cpu(), self.table.cpu()
        assert self.lens.tolist() == [len(x) for x in self.keys]
        for n, x in enumerate(self.keys):
            pos = torch.arange(len(x))
            held = table[n, pos // PAGE].long(), pos % PAGE
            want, err = turned(x, pos, self.freq, False)
            within(kc[held], want, err, self.dtype, R)
            assert torch.equal(vc[held], self.values[n])
        return q

    def check(self, q, got, cu=None, window=None, sinks=0):
        def seen(pos, j):
            return (j <= pos) if window is None else (j > pos - window) | (j < sinks)

        lens, c = self.lens.cpu(), q.cpu()
        want = attention(c, self.pool[0].cpu(), self.pool[1].cpu(), self.table.cpu(), lens, D ** -0.5, seen,
                         None if cu is None else cu.cpu())
        assert not misses(*got, want, c, lens.tolist(), D ** -0.5, cu)

    def args(self, q):
        return q, self.pool[0], self.pool[1], self.table, self.lens

    def fork(self, src, dst):
        paged_free(self.table, self.lens, self.refs, self.i32(dst))
        assert bool(paged_fork(self.pool, self.table, self.lens, self.refs, self.i32(src), self.i32(dst)).all())
        for s, d in zip(src, dst):
            self.keys[d], self.values[d] = self.keys[s], self.values[s]

    def free(self, rows):
        paged_free(self.table, self.lens, self.refs, self.i32(rows))
        for n in rows:
            self.keys[n], self.values[n] = self.keys[n][:0], self.values[n][:0]

    def compact(self):
        self.table, self.refs, _ = paged_compact(self.pool, self.table, self.refs)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("width", [30, 9000])  # shared tokens looked at one by one, and together
def test_answers_to_prompts(dtype, width, gpu_device):
    each, prompts = 5, [37, 150, 64]
    loop = Loop(gpu_device, each * 3, 120, width, dtype, seed=width)
    new = [0] * (each * 3)
    for g, n in enumerate(prompts):
        new[g * each] = n
    cu = loop.i32([0] + new).cumsum(0, dtype=torch.int32)
    q = loop.append(new, cu)
    loop.check(q, paged_attention(*loop.args(q), cu_seqlens=cu, return_lse=True), cu)
    for g in range(3):
        loop.fork([g * each] * (each - 1), list(range(g * each + 1, (g + 1) * each)))
    groups, shared = loop.i32([0, each, 2 * each, 3 * each]), loop.i32(prompts)
    for step in range(8):
        if step == 3:  # two answers end, the first of its group among them; their pages are others'
            loop.free([5, 12])
            loop.compact()
        live = [int(n > 0) for n in loop.lens.tolist()]
        # (rows that have ended: no tokens)
        cu = loop.i32([0] + live).cumsum(0, dtype=torch.int32)
        q = loop.append(live, cu)
        loop.check(q, paged_attention_shared(*loop.args(q), groups, shared, cu_seqlens=cu, return_lse=True), cu)
    # a draft of 4 tokens for every answer, three of them rejected
    loop.free(list(range(10, 15)))
    loop.fork([6], [5])
    q = loop.append([4] * 10 + [0] * 5, loop.i32(list(range(0, 41, 4)) + [40] * 5))
    cu = loop.i32(list(range(0, 41, 4)) + [40] * 5)
    loop.check(q, paged_attention_shared(*loop.args(q), groups, shared, cu_seqlens=cu, return_lse=True), cu)
    loop.lens[:10] -= 3
    loop.keys = [x[:len(x) - 3] for x in loop.keys[:10]] + loop.keys[10:]
    loop.values = [x[:len(x) - 3] for x in loop.values[:10]] + loop.values[10:]
    q = loop.append([1] * 10 + [0] * 5, loop.i32(list(range(11)) + [10] * 5))
    cu = loop.i32(list(range(11)) + [10] * 5)
    for window, sinks in ((20, 4), (50, 33)):
        loop.check(q, paged_attention(*loop.args(q), window=window, sinks=sinks, cu_seqlens=cu, return_lse=True), cu,
                   window, sinks)


def test_a_stream_gives_its_pages_away(gpu_device):
    """A row under a window with first tokens: pages between them are another
    row's before long."""
    loop = Loop(gpu_device, 2, 24, 40, torch.bfloat16, seed=3)
    window, sinks = 64, 20
    q = loop.append([100, 0], loop.i32([0, 100, 100]))
    for step in range(6):
        q = loop.append([30, 0], loop.i32([0, 30, 30]))
        cu = loop.i32([0, 30, 30])
        got = paged_attention(*loop.args(q), window=window, sinks=sinks, cu_seqlens=cu, return_lse=True)
        loop.check(q, got, cu, window, sinks)
        # what is behind the first tokens' pages and before the window of the next chunk
        first, last = -(-sinks // PAGE), (int(loop.lens[0]) + 1 - window) // PAGE
        kept = loop.table.clone()
        gone = loop.table[0, first:last].clone()
        loop.pool[:, gone[gone >= 0].long()] = float("nan")
        loop.table[0, first:last] = -1
        q = torch.randn(2, 1, HQ, D, generator=loop.gen).to(torch.bfloat16).to(gpu_device)
        o, lse = paged_attention(*loop.args(q), window=window, sinks=sinks, return_lse=True)
        want = attention(q.cpu(), loop.pool[0].cpu(), loop.pool[1].cpu(), loop.table.cpu(), loop.lens.cpu(), D ** -0.5,
                         lambda pos, j: (j > pos - window) | (j < sinks))
        assert not misses(o, lse, want, q.cpu(), loop.lens.tolist(), D ** -0.5)
        # (the test's own record goes on from whole pages)
        loop.table = kept
        for n, x in enumerate(loop.keys):
            pos = torch.arange(len(x))
            held = kept[n].cpu()[pos // PAGE].long(), pos % PAGE
            want, _ = turned(x, pos, loop.freq, False)
            k, v = loop.pool[0].cpu(), loop.pool[1].cpu()
            k[held], v[held] = want.to(torch.bfloat16), loop.values[n]
            loop.pool[0].copy_(k)
            loop.pool[1].copy_(v)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_pages_given_away_are_another_rows(dtype, gpu_device):
    """A row under a window with first tokens hands the pages between the two back
    (filled with NaN), another one's next tokens go into them, and both go on: more
    tokens altogether than the pool has places for."""
    d, gen = gpu_device, torch.Generator().manual_seed(4)
    window, sinks, pages, width = 64, 20, 24, 32
    i32 = dict(dtype=torch.int32, device=d)
    pool = torch.full((2, pages, PAGE, HKV, D), float("nan"), dtype=dtype, device=d)
    table, lens, refs = torch.full((2, width), -1, **i32), torch.zeros(2, **i32), torch.zeros(pages, **i32)
    # what the rows hold, on the CPU, each in pages of its own one after the other
    rows = torch.zeros(2, 2 * width, PAGE, HKV, D, dtype=dtype)
    own = torch.arange(2 * width, dtype=torch.int32).view(2, width)
    given, total = set(), [0, 0]
    for new in ([100, 3], [30, 40], [30, 41], [30, 40], [1, 40], [30, 37], [33, 1], [7, 40]):
        assert bool(paged_reserve(table, lens, refs, torch.tensor(new, **i32), PAGE).all())
        cu = torch.tensor([0, new[0], sum(new)], **i32)
        q, k, v = torch.randn(1, sum(new), HQ + 2 * HKV, D, generator=gen).clamp(-6, 6).to(dtype).split([HQ, HKV, HKV], 2)
        paged_append(k.to(d), v.to(d), pool[0], pool[1], table, lens, cu_seqlens=cu)
        for n, first in enumerate((0, new[0])):
            pos = torch.arange(total[n], total[n] + new[n])
            for c, x in zip(rows, (k, v)):
                c[own[n, pos // PAGE].long(), pos % PAGE] = x[0, first:first + new[n]]
            total[n] += new[n]
        assert lens.tolist() == total
        got = paged_attention(q.to(d), pool[0], pool[1], table, lens, window=window, sinks=sinks, cu_seqlens=cu, return_lse=True)
        want = attention(q, rows[0], rows[1], own, total, D ** -0.5, lambda pos, j: (j > pos - window) | (j < sinks), cu.cpu())
        assert not misses(*got, want, q, total, D ** -0.5, cu.cpu())
        for n in range(2):
            gone = table[n, -(-sinks // PAGE):max(0, (total[n] + 1 - window) // PAGE)]
            at = gone[gone >= 0].long()
            given |= {(n, p) for p in at.tolist()}
            pool[:, at] = float("nan")
            refs[at] -= 1
            gone[:] = -1
    held = {(n, p) for n in range(2) for p in table[n].tolist() if p >= 0}
    assert {(1 - n, p) for n, p in given} & held and sum(total) > pages * PAGE
