"""The paged cache's operators in plain form, on the CPU: attention in 64 bits
from its definition, one query at a time; the page operations as loops over
lists.  Test infrastructure only."""

from __future__ import annotations

import math

import torch


def spans(N, T, cu=None):
    """(first token index, new tokens) of each sequence in the flattened tokens."""
    if cu is None:
        return [(n * T, T) for n in range(N)]
    c = [int(x) for x in cu]
    return [(c[n], c[n + 1] - c[n]) for n in range(N)]


def cached(cache, table, n, length, h):
    """The first ``length`` rows of head h of sequence n, fp64 [length, D]."""
    size, D = cache.shape[1], cache.shape[3]
    if length == 0:
        return torch.zeros(0, D, dtype=torch.float64)
    pages = [int(table[n, j]) for j in range(-(-length // size))]
    return torch.cat([cache[p, :, h].double() for p in pages])[:length]


def attention(q, k_cache, v_cache, table, lens, scale, causal=True, window=None, cu=None):
    """(o, lse) in fp64, in the shapes of the call's."""
    B, T, HQ, D = q.shape
    N, HKV = table.shape[0], k_cache.shape[2]
    G = HQ // HKV
    qf = q.reshape(B * T, HQ, D).double()
    o = torch.zeros(B * T, HQ, D, dtype=torch.float64)
    lse = torch.full((B * T, HQ), -math.inf, dtype=torch.float64)
    for n, (first, count) in enumerate(spans(N, T, cu)):
        L = int(lens[n])
        j = torch.arange(L)
        pos = torch.arange(L - count, L)[:, None]
        seen = torch.ones(count, L, dtype=torch.bool)
        if causal:
            seen &= j <= pos
        if window:
            seen &= j > pos - window
        for h in range(HKV):
            K, V = cached(k_cache, table, n, L, h), cached(v_cache, table, n, L, h)
            for g in range(h * G, (h + 1) * G):
                x = scale * (qf[first:first + count, g] @ K.t())
                x = x.masked_fill(~seen, -math.inf)
                z = torch.logsumexp(x, 1) if L else torch.full((count,), -math.inf, dtype=torch.float64)
                some = torch.isfinite(z)
                w = torch.where(some[:, None], torch.exp(x - torch.where(some, z, torch.zeros_like(z))[:, None]),
                                torch.zeros_like(x))
                o[first:first + count, g] = w @ V
                lse[first:first + count, g] = z
    return o.view(q.shape), lse.view(B, T, HQ)


def append(k, v, k_cache, v_cache, table, lens, cu=None):
    size, N = k_cache.shape[1], table.shape[0]
    kf, vf = k.reshape(-1, *k.shape[2:]), v.reshape(-1, *v.shape[2:])
    for n, (first, count) in enumerate(spans(N, k.shape[1], cu)):
        for i in range(count):
            pos = int(lens[n]) - count + i
            if pos < 0 or pos // size >= table.shape[1]:
                continue
            page = int(table[n, pos // size])
            if 0 <= page < k_cache.shape[0]:
                k_cache[page, pos % size] = kf[first + i]
                v_cache[page, pos % size] = vf[first + i]


def _free_pages(refs):
    return [p for p, r in enumerate(refs) if r == 0]


def reserve(table, lens, refs, more, size):
    """In place on lists (table: a list of rows); the ok list."""
    free, at, ok = _free_pages(refs), 0, []
    for n in range(len(lens)):
        have, want = -(-lens[n] // size), -(-(lens[n] + max(0, more[n])) // size)
        if want > len(table[n]):
            ok.append(False)
            continue
        need = max(0, want - have)
        got = free[at:at + need]
        at += need
        ok.append(len(got) == need)
        if ok[-1]:
            for i, p in enumerate(got):
                table[n][have + i] = p
                refs[p] = 1
            lens[n] += max(0, more[n])
    return ok


def free(table, lens, refs, rows):
    for n in rows:
        if 0 <= n < len(lens):
            for j, p in enumerate(table[n]):
                if 0 <= p < len(refs):
                    refs[p] -= 1
                table[n][j] = -1
            lens[n] = 0


def fork(pools, table, lens, refs, src, dst, size):
    """``pools`` are tensors [lead, P, ...] changed in place; the ok list."""
    free_, at, ok, taken = _free_pages(refs), 0, [], []
    for s, d in zip(src, dst):
        full, part = lens[s] // size, lens[s] % size > 0
        page = None
        if part:
            page = free_[at] if at < len(free_) else None
            at += 1
        if part and page is None:
            ok.append(False)
            continue
        ok.append(True)
        for j in range(len(table[d])):
            table[d][j] = table[s][j] if j < full else -1
            if j < full:
                refs[table[s][j]] += 1
        if part:
            taken.append((table[s][full], page))
            table[d][full] = page
        lens[d] = lens[s]
    for old, new in taken:
        refs[new] = 1
        for t in pools:
            t[:, new] = t[:, old]
    return ok


def compact(pools, table, refs):
    """(table, refs, live); ``pools`` changed in place."""
    live = sum(1 for r in refs if r)
    holes = [p for p in range(live) if refs[p] == 0]
    movers = [p for p in range(live, len(refs)) if refs[p]]
    to = dict(zip(movers, holes))
    for old, new in to.items():
        for t in pools:
            t[:, new] = t[:, old]
    new_refs = [0 if p in to else r for p, r in enumerate(refs)]
    for old, new in to.items():
        new_refs[new] = refs[old]
    return [[to.get(p, p) for p in row] for row in table], new_refs, live
