"""Attention over a paged cache in 64 bits for any rule of what a query sees,
one sequence and head at a time, on the CPU; and caches for its tests.  Test
infrastructure only."""

from __future__ import annotations

import math

import torch

from paged_oracle import spans


def attention(q, k_cache, v_cache, table, lens, scale, seen, cu=None):
    """(o, lse, sum of w |v|) in fp64, in the shapes of the call's.
    ``seen(pos, j)``: whether the query at pos sees key j (tensors); entries of
    the table that are no page are keys that nobody sees."""
    B, T, HQ, D = q.shape
    N, HKV, size = table.shape[0], k_cache.shape[2], k_cache.shape[1]
    G = HQ // HKV
    qf = q.reshape(B * T, HQ, D).double()
    o = torch.zeros(B * T, HQ, D, dtype=torch.float64)
    mass = torch.zeros_like(o)
    lse = torch.full((B * T, HQ), -math.inf, dtype=torch.float64)
    for n, (first, count) in enumerate(spans(N, T, cu)):
        L = int(lens[n])
        if L == 0 or count == 0:
            continue
        pos, j = torch.arange(L - count, L)[:, None], torch.arange(L)
        see = seen(pos, j) & (j <= pos)
        some = see.any(0)  # (what nobody sees may be anything)
        keys = j[some]
        at = table[n, keys // size].long()
        assert bool((at >= 0).all())
        see = see[:, some].repeat_interleave(G, 0)
        for h in range(HKV):
            K, V = (c[at, keys % size, h].double() for c in (k_cache, v_cache))
            x = scale * (qf[first:first + count, h * G:(h + 1) * G].reshape(count * G, D) @ K.t())
            x = x.masked_fill(~see, -math.inf)
            z = torch.logsumexp(x, 1)
            w = torch.exp(x - torch.where(torch.isfinite(z), z, torch.zeros_like(z))[:, None])
            w = w.masked_fill(~see, 0.0)
            o[first:first + count, h * G:(h + 1) * G] = (w @ V).view(count, G, D)
            mass[first:first + count, h * G:(h + 1) * G] = (w @ V.abs()).view(count, G, D)
            lse[first:first + count, h * G:(h + 1) * G] = z.view(count, G)
    return o.view(q.shape), lse.view(B, T, HQ), mass.view(q.shape)


def on_device(cache, dev):
    """The cache on the GPU, in the layout that it has."""
    if cache.is_contiguous():
        return cache.to(dev)
    return cache.transpose(1, 2).contiguous().to(dev).transpose(1, 2)


def caches(table, P, HKV, D, page, dtype, held, gen, layout="token"):
    """Keys and values of unit variance where ``held [P, page]`` says so, NaN
    everywhere else."""
    out = []
    for _ in range(2):
        c = torch.randn((P, HKV, page, D) if layout == "head" else (P, page, HKV, D), generator=gen).clamp(-6, 6).to(dtype)
        c = c.transpose(1, 2) if layout == "head" else c
        c[~held] = math.nan
        out.append(c)
    return out


def tables(lens, page, gen, width=0, spare=2):
    need = [-(-n // page) for n in lens]
    P = sum(need) + spare
    order = torch.randperm(P, generator=gen, dtype=torch.int32)
    table = torch.full((len(lens), max(need + [1, width])), -1, dtype=torch.int32)
    at = 0
    for n, c in enumerate(need):
        table[n, :c] = order[at:at + c]
        at += c
    return table, P


def held_tokens(table, P, lens, page, gone=lambda n, j: False):
    """Which places hold a sequence's token (those ``gone`` excepted)."""
    held = torch.zeros(P, page, dtype=torch.bool)
    for n, L in enumerate(lens):
        for j in range(L):
            if not gone(n, j):
                held[int(table[n, j // page]), j % page] = True
    return held
