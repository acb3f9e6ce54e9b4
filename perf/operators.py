"""Attention over a paged cache of keys and values, and the work on its pages, as cases to time and to compare.

A cache is a pool of pages of ``page`` tokens, ``[P, page, HKV, D]`` for the
keys and for the values of a layer.  ``page_table [N, M]`` names the pages
of each sequence (-1: none), ``seq_lens [N]`` counts its cached tokens (new
ones included) and ``page_refs [P]`` the sequences that hold each page.

A case is a dict of plain values.  ``op`` is

* ``attention``: new tokens of each sequence over its cached ones (causal);
* ``append``: new keys and values into their places in the pages;
* ``beam``: rows freed, others forked into them, room reserved in them;
* ``compact``: live pages moved down until they are the pool's first;
* ``copy``: rows of a pool copied to others.

Lengths are spread by a seed of the case's own (``spread``), so that they
belong to the case; values come from the seed that ``prepare`` is given.
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False


def _attention(name, N, T, lo, hi, HQ, HKV, D=128, page=16, dtype="bf16", packed=False, window=0, lse=False,
               layout="token", spread=1):
    return {"name": name, "op": "attention", "N": N, "T": T, "lo": lo, "hi": hi, "HQ": HQ, "HKV": HKV, "D": D,
            "page": page, "dtype": dtype, "packed": packed, "window": window, "lse": lse, "layout": layout,
            "spread": spread}


def _append(name, N, T, lo, hi, HKV, D=128, page=16, dtype="bf16", packed=False, layout="token", spread=1):
    return {"name": name, "op": "append", "N": N, "T": T, "lo": lo, "hi": hi, "HKV": HKV, "D": D, "page": page,
            "dtype": dtype, "packed": packed, "layout": layout, "spread": spread}


def _beam(name, N, F, lo, hi, layers, HKV, D=128, page=16, grow=1, spread=1):
    return {"name": name, "op": "beam", "N": N, "F": F, "lo": lo, "hi": hi, "layers": layers, "HKV": HKV, "D": D,
            "page": page, "grow": grow, "spread": spread}


def _compact(name, P, N, live, layers, HKV, D=128, page=16, spread=1):
    return {"name": name, "op": "compact", "P": P, "N": N, "live": live, "layers": layers, "HKV": HKV, "D": D,
            "page": page, "spread": spread}


def _copy(name, layers, rows, count, H, a, b, dtype="f32"):
    return {"name": name, "op": "copy", "layers": layers, "rows": rows, "count": count, "H": H, "a": a, "b": b,
            "dtype": dtype}


def listed():
    return [
        # One decode step of one short conversation: the smallest call, where
        # latency counts.
        _attention("decode_1x700", 1, 1, 700, 700, 32, 8),
        # One decode step of a full serving batch, conversations of 100 to
        # 16000 tokens: the cache streamed once.
        _attention("decode_64_ragged", 64, 1, 100, 16000, 32, 8, layout="head"),
        # A draft of 5 tokens to verify in each of 16 sequences; fp16, small
        # heads in groups of 6.
        _attention("draft_16x5_fp16_d64", 16, 5, 333, 8191, 24, 4, D=64, page=32, dtype="fp16"),
        # A packed batch of a serving step: prompt chunks of uneven lengths
        # after contexts of up to 12000 tokens, single tokens among them, a
        # sliding window of 4096; with the log-sum-exp.
        _attention("chunk_packed8_window", 8, 1024, 900, 12000, 32, 8, page=64, packed=True, window=4096, lse=True),
        # One long prompt into an empty cache: the largest attention.
        _attention("prefill_1x8192", 1, 8192, 8192, 8192, 32, 8),
        # The new token of each of 128 sequences.
        _append("append_128x1", 128, 1, 100, 8000, 8),
        # 16 prompts of uneven lengths, packed.
        _append("append_packed16_t1024", 16, 1024, 1024, 6000, 8, packed=True, layout="head"),
        # A beam search step: 8 prompts of 4 beams, half of the beams replaced.
        _beam("beam_32_fork16", 32, 16, 700, 4000, 4, 8),
        # 63 answers forked from the row of a prompt, one cache for 16 layers.
        _beam("beam_64_fork63", 64, 63, 8000, 8191, 16, 8, grow=40),
        # A small pool, a third free.
        _compact("compact_256", 256, 12, 0.66, 2, 8),
        # A pool of 16 layers, half of it free: the largest move.
        _compact("compact_2048", 2048, 24, 0.5, 16, 8),
        # The recurrent states of 12 layers forked along with their sequences.
        _copy("copy_states_8_of_48", 12, 48, 8, 32, 128, 128),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["decode", "decode", "draft", "chunk", "chunk", "prefill", "append", "append", "beam", "compact",
                     "copy"])
    spread = rng.randrange(1, 1 << 20)
    HKV = rng.choice([1, 2, 4, 8])
    D = rng.choice([64, 128, 128])
    page = rng.choice([16, 16, 32, 64, 128])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    layout = rng.choice(["token", "head"])
    kw = {"D": D, "page": page, "dtype": dtype, "layout": layout, "spread": spread}
    if op in ("decode", "draft", "chunk", "prefill"):
        HQ = HKV * rng.choice([1, 2, 4, 6, 8])
        kw["window"] = rng.choice([0, 0, 0, _log_int(rng, 100, 4096)])
        kw["lse"] = rng.random() < 0.3
    if op in ("decode", "draft"):
        T = 1 if op == "decode" else rng.randint(2, 8)
        N = _log_int(rng, 1, 128)
        lo = _log_int(rng, max(T, 20), 2000)
        hi = _log_int(rng, lo, max(lo, min(32000, 64 * 16000 // N)))
        return _unnamed(_attention("", N, T, lo, hi, HQ, HKV, **kw))
    if op == "chunk":
        # padded queries times keys times heads: the scores of the plain form
        N, T = rng.randint(1, 8), _log_int(rng, 20, 1024)
        lo = _log_int(rng, T, 4000)
        hi = min(_log_int(rng, lo, 12000), max(lo, 8 * 1024 * 32 * 12000 // (N * T * HQ)))
        return _unnamed(_attention("", N, T, lo, hi, HQ, HKV, packed=rng.random() < 0.7, **kw))
    if op == "prefill":
        T = _log_int(rng, 1000, 8192)
        HQ = min(HQ, 32)
        HKV = HKV if HQ % HKV == 0 else 1
        return _unnamed(_attention("", 1, T, T, T + rng.choice([0, 0, rng.randint(0, T // 4)]) if T < 6000 else T,
                                   HQ, HKV, **kw))
    if op == "append":
        N, T = _log_int(rng, 1, 128), _log_int(rng, 1, 1024)
        T = min(T, 16 * 1024 // N)
        lo = _log_int(rng, max(T, 50), 4000)
        return _unnamed(_append("", N, T, lo, _log_int(rng, lo, 8000), HKV, packed=rng.random() < 0.6, **kw))
    if op == "beam":
        N = rng.randint(2, 64)
        lo = _log_int(rng, 50, 4000)
        return _unnamed(_beam("", N, rng.randint(1, N - 1), lo, min(8191, _log_int(rng, lo, 8191)),
                              rng.randint(1, 16), HKV, D=D, page=page, grow=_log_int(rng, 1, 100), spread=spread))
    if op == "compact":
        page = min(page, 64)
        P = max(32, _log_int(rng, 64, 2048) * 16 // page)
        return _unnamed(_compact("", P, rng.randint(2, 32), round(rng.uniform(0.2, 0.95), 2), rng.randint(1, 16),
                                 HKV, D=D, page=page, spread=spread))
    rows = rng.randint(4, 48)
    H, a = rng.choice([4, 8, 16, 32]), rng.choice([16, 64, 128])
    return _unnamed(_copy("", rng.randint(1, 12), rows, rng.randint(1, max(1, min(8, rows // 2))), H, a, 128,
                          dtype=rng.choice(["f32", "bf16"])))


def _unnamed(case):
    return {k: v for k, v in case.items() if k != "name"}


# -- lengths and tables ---------------------------------------------------


def _lengths(case):
    """(cached tokens, new tokens) of each sequence: the cached ones spread by
    their logarithm between lo and hi, in packed batches the new ones from a
    single token up to T (the last sequence's T)."""
    rng = random.Random(case["spread"])
    lens = [_log_int(rng, case["lo"], case["hi"]) for _ in range(case["N"])]
    T = case.get("T", 0)
    new = [T] * case["N"]
    if case.get("packed"):
        new = [1 if rng.random() < 0.35 else _log_int(rng, 1, T) for _ in lens[:-1]] + [T]
    return lens, new


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}


def _table(lens, page, gen, spare=0, width=0):
    """A page table of pages in no order, and the number of pages of its pool."""
    need = [-(-n // page) for n in lens]
    P = sum(need) + spare
    order = torch.randperm(P, generator=gen, device="cuda", dtype=torch.int32)
    M = max(max(need), width)
    at = torch.tensor(need, device="cuda")
    start = torch.cumsum(at, 0) - at
    col = torch.arange(M, device="cuda")
    idx = (start[:, None] + col).clamp_(max=P - 1)
    table = torch.where(col < at[:, None], order[idx], torch.full_like(idx, -1, dtype=torch.int32))
    return table.contiguous(), P


def _randn(gen, dtype, *shape):
    out = torch.empty(shape, dtype=dtype, device="cuda")
    return out.normal_(generator=gen)


def _cache(case, P, gen):
    """Keys and values [P, page, HKV, D]; in the "head" layout a view of
    [P, HKV, page, D], the tokens of a head in one piece."""
    dt, page, H, D = _DTYPES[case["dtype"]], case["page"], case["HKV"], case["D"]
    if case["layout"] == "head":
        return [_randn(gen, dt, P, H, page, D).transpose(1, 2) for _ in range(2)]
    return [_randn(gen, dt, P, page, H, D) for _ in range(2)]


def _cu(new):
    return torch.tensor([0] + new, dtype=torch.int32, device="cuda").cumsum(0, dtype=torch.int32)


# -- prepare --------------------------------------------------------------


def prepare(case, seed):
    gen = _gen(seed)
    return {"attention": _prepare_attention, "append": _prepare_append, "beam": _prepare_beam,
            "compact": _prepare_compact, "copy": _prepare_copy}[case["op"]](case, gen) | {"case": case}


def _prepare_attention(case, gen):
    lens, new = _lengths(case)
    table, P = _table(lens, case["page"], gen, spare=3)
    k, v = _cache(case, P, gen)
    dt, HQ, D = _DTYPES[case["dtype"]], case["HQ"], case["D"]
    shape = (1, sum(new)) if case["packed"] else (case["N"], case["T"])
    return {"q": _randn(gen, dt, *shape, HQ, D), "k": k, "v": v, "table": table,
            "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "cu": _cu(new) if case["packed"] else None,
            "scale": D ** -0.5, "window": case["window"] or None, "tmax": max(new)}


def _prepare_append(case, gen):
    lens, new = _lengths(case)
    table, P = _table(lens, case["page"], gen, spare=3)
    k, v = _cache(case, P, gen)
    dt, H, D = _DTYPES[case["dtype"]], case["HKV"], case["D"]
    shape = (1, sum(new)) if case["packed"] else (case["N"], case["T"])
    # keys and values as a fused projection leaves them, side by side
    kv = _randn(gen, dt, *shape, 2 * H, D)
    return {"new_k": kv[:, :, :H], "new_v": kv[:, :, H:], "k": k, "v": v, "table": table,
            "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "cu": _cu(new) if case["packed"] else None}


def _prepare_beam(case, gen):
    lens, _ = _lengths(case)
    page, N, F, grow = case["page"], case["N"], case["F"], case["grow"]
    width = -(-(max(lens) + grow) // page)
    table, P = _table(lens, page, gen, spare=F * (2 + grow // page), width=width)
    refs = torch.zeros(P, dtype=torch.int32, device="cuda")
    held = table[table >= 0].long()
    refs.index_add_(0, held, torch.ones_like(held, dtype=torch.int32))
    # the rows to replace, and for each a row that stays
    rows = torch.randperm(N, generator=gen, device="cuda", dtype=torch.int32)
    dst, stay = rows[:F].contiguous(), rows[F:]
    pick = torch.randint(0, N - F, (F,), generator=gen, device="cuda")
    more = torch.zeros(N, dtype=torch.int32, device="cuda")
    more[dst.long()] = grow
    pool = _randn(gen, torch.bfloat16, case["layers"], 2, P, page, case["HKV"], case["D"])
    return {"pool": pool, "table": table, "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "refs": refs,
            "src": stay[pick].contiguous(), "dst": dst, "more": more}


def _compact_lens(case):
    """Lengths whose pages are the live share of the pool."""
    rng = random.Random(case["spread"])
    pages = max(case["N"], int(case["P"] * case["live"]))
    cuts = sorted(rng.sample(range(1, pages), case["N"] - 1)) if pages > case["N"] else list(range(1, case["N"]))
    return [(b - a) * case["page"] - rng.randrange(case["page"]) for a, b in zip([0] + cuts, cuts + [pages])]


def _prepare_compact(case, gen):
    lens = _compact_lens(case)
    used = sum(-(-n // case["page"]) for n in lens)
    table, P = _table(lens, case["page"], gen, spare=max(0, case["P"] - used))
    refs = torch.zeros(P, dtype=torch.int32, device="cuda")
    held = table[table >= 0].long()
    refs.index_add_(0, held, torch.ones_like(held, dtype=torch.int32))
    pool = _randn(gen, torch.bfloat16, case["layers"], 2, P, case["page"], case["HKV"], case["D"])
    return {"pool": pool, "table": table, "refs": refs}


def _prepare_copy(case, gen):
    pool = _randn(gen, _DTYPES[case["dtype"]], case["layers"], case["rows"], case["H"], case["a"], case["b"])
    order = torch.randperm(case["rows"], generator=gen, device="cuda", dtype=torch.int32)
    n = case["count"]
    return {"pool": pool, "src": order[:n].contiguous(), "dst": order[n:2 * n].contiguous()}


# -- run ------------------------------------------------------------------


def _bits(t):
    """A tensor's values as whole numbers, for what is only moved."""
    return t.view(torch.int16 if t.element_size() == 2 else torch.int32)


def run(state):
    op = state["case"]["op"]
    if own:
        return {"attention": _own_attention, "append": _own_append, "beam": _own_beam, "compact": _own_compact,
                "copy": _own_copy}[op](state)
    return {"attention": _plain_attention, "append": _plain_append, "beam": _plain_beam, "compact": _plain_compact,
            "copy": _plain_copy}[op](state)


def _package():
    path = os.path.join(os.getcwd(), "kda-ascendc_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import kda_bt16

    return kda_bt16


def _own_attention(s):
    lse = s["case"]["lse"]
    r = _package().paged_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], scale=s["scale"], window=s["window"],
                                   cu_seqlens=s["cu"], return_lse=lse)
    return {"o": r[0], "lse": r[1]} if lse else {"o": r}


def _own_append(s):
    _package().paged_append(s["new_k"], s["new_v"], s["k"], s["v"], s["table"], s["lens"], cu_seqlens=s["cu"])
    return {"k": _bits(s["k"]), "v": _bits(s["v"])}


def _own_beam(s):
    kda = _package()
    kda.paged_free(s["table"], s["lens"], s["refs"], s["dst"])
    forked = kda.paged_fork(s["pool"], s["table"], s["lens"], s["refs"], s["src"], s["dst"])
    grown = kda.paged_reserve(s["table"], s["lens"], s["refs"], s["more"], s["case"]["page"])
    return {"table": s["table"], "lens": s["lens"], "refs": s["refs"], "forked": forked, "grown": grown,
            "pool": _bits(s["pool"])}


def _own_compact(s):
    table, refs, live = _package().paged_compact(s["pool"], s["table"], s["refs"])
    return {"table": table, "refs": refs, "live": live, "pool": _bits(s["pool"])}


def _own_copy(s):
    _package().paged_copy(s["pool"], s["src"], s["dst"])
    return {"pool": _bits(s["pool"])}


def _places(s, tokens):
    """(sequence, position in it) of each new token, in the order of q."""
    lens = s["lens"].long()
    i = torch.arange(tokens, device=lens.device)
    if s["cu"] is None:
        T = s["case"]["T"]
        return i // T, lens[i // T] - T + i % T
    cu = s["cu"].long()
    n = torch.searchsorted(cu, i, right=True) - 1
    return n, lens[n] - cu[n + 1] + i


def _plain_attention(s):
    q, k, v, table, lens = s["q"], s["k"], s["v"], s["table"].long(), s["lens"].long()
    N, M = table.shape
    page, HKV, D = k.shape[1:]
    HQ = q.shape[2]
    G, T = HQ // HKV, s["tmax"]
    tokens = q.shape[0] * q.shape[1]
    n, pos = _places(s, tokens)
    row = pos - lens[n] + T  # the last new token of a sequence at row T - 1
    qp = torch.zeros(N, T, HQ, D, dtype=torch.float32, device=q.device)
    qp[n, row] = q.reshape(tokens, HQ, D).float()
    qp = qp.view(N, T, HKV, G, D).permute(0, 2, 3, 1, 4).reshape(N, HKV, G * T, D)
    pages = table.clamp(min=0)
    kk = k[pages].float().reshape(N, M * page, HKV, D).permute(0, 2, 3, 1).contiguous()
    vv = v[pages].float().reshape(N, M * page, HKV, D).permute(0, 2, 1, 3).contiguous()
    x = torch.matmul(qp, kk).mul_(s["scale"]).view(N, HKV, G, T, M * page)
    j = torch.arange(M * page, device=q.device)
    at = (lens[:, None] - T + torch.arange(T, device=q.device))[:, :, None]
    hide = (j > at) | (j >= lens[:, None, None])
    if s["window"]:
        hide |= j <= at - s["window"]
    x.masked_fill_(hide[:, None, None], float("-inf"))
    # keys of no sequence: whatever the pages hold there
    vv.masked_fill_((j >= lens[:, None])[:, None, :, None], 0.0)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(N, HKV, G * T, M * page), vv).view(N, HKV, G, T, D)
    o = o / torch.where(total > 0, total, torch.ones_like(total))
    o = o.permute(0, 3, 1, 2, 4).reshape(N, T, HQ, D)[n, row].view(q.shape).to(q.dtype)
    if not s["case"]["lse"]:
        return {"o": o}
    lse = (top + total.log()).squeeze(-1).permute(0, 3, 1, 2).reshape(N, T, HQ)[n, row]
    return {"o": o, "lse": lse.view(q.shape[:3])}


def _plain_append(s):
    nk, nv = s["new_k"], s["new_v"]
    tokens = nk.shape[0] * nk.shape[1]
    n, pos = _places(s, tokens)
    page = s["k"].shape[1]
    at = s["table"].long()[n, pos // page]
    s["k"][at, pos % page] = nk.reshape(tokens, *nk.shape[2:])
    s["v"][at, pos % page] = nv.reshape(tokens, *nv.shape[2:])
    return {"k": _bits(s["k"]), "v": _bits(s["v"])}


def _free_pages(refs):
    """The free pages in rising order, then the others; and their number."""
    return torch.sort((refs != 0).to(torch.uint8), stable=True).indices, (refs == 0).sum()


def _count(refs, pages, by):
    """refs += by for each page named (-1: none)."""
    refs.index_add_(0, pages.clamp(min=0).reshape(-1).long(), ((pages >= 0) * by).reshape(-1).to(torch.int32))


def _plain_beam(s):
    pool, table, lens, refs, src, dst = s["pool"], s["table"], s["lens"], s["refs"], s["src"].long(), s["dst"].long()
    page, M = pool.shape[3], table.shape[1]
    col = torch.arange(M, device=table.device)
    # free
    _count(refs, table[dst], -1)
    table[dst] = -1
    lens[dst] = 0
    # fork: whole pages shared, the last one's tokens copied to a page of their own
    n = lens[src].long()
    full, part = n // page, n % page > 0
    order, have = _free_pages(refs)
    rank = torch.cumsum(part, 0) - 1
    forked = ~part | (rank < have)
    fresh = order[rank.clamp(0, refs.numel() - 1)]
    rows = table[src]
    last = rows.gather(1, full.clamp(max=M - 1)[:, None]).squeeze(1).long()
    shared = torch.where((col < full[:, None]) & forked[:, None], rows, torch.full_like(rows, -1))
    _count(refs, shared, 1)
    take = part & forked
    _count(refs, torch.where(take, fresh, torch.full_like(fresh, -1)), 1)
    table[dst] = torch.where((col == full[:, None]) & take[:, None], fresh[:, None].to(torch.int32), shared)
    lens[dst] = torch.where(forked, lens[src], torch.zeros_like(lens[src]))
    took, whence = fresh[take], last[take]
    pool[:, :, took] = pool[:, :, whence]
    # reserve
    more = s["more"]
    have_pages = (lens + (page - 1)) // page
    want = (lens + more + (page - 1)) // page
    need = (want - have_pages).long()
    order, have = _free_pages(refs)
    end = torch.cumsum(need, 0)
    grown = (need == 0) | (end <= have)
    nth = (end - need)[:, None] + (col - have_pages[:, None])
    new = (col >= have_pages[:, None]) & (col < want[:, None]) & grown[:, None]
    pages = order[nth.clamp(0, refs.numel() - 1)].to(torch.int32)
    table.copy_(torch.where(new, pages, table))
    _count(refs, torch.where(new, pages, torch.full_like(pages, -1)), 1)
    lens += torch.where(grown, more, torch.zeros_like(more))
    return {"table": table, "lens": lens, "refs": refs, "forked": forked, "grown": grown, "pool": _bits(pool)}


def _plain_compact(s):
    pool, table, refs = s["pool"], s["table"], s["refs"]
    P = refs.numel()
    used = refs != 0
    live = used.sum()
    page = torch.arange(P, device=refs.device)
    holes, movers = page[~used & (page < live)], page[used & (page >= live)]
    to = page.clone()
    to[movers] = holes
    pool[:, :, holes] = pool[:, :, movers]
    table = torch.where(table >= 0, to[table.clamp(min=0).long()].to(torch.int32), table)
    refs = refs.clone()
    refs[holes] = refs[movers]
    refs[movers] = 0
    return {"table": table, "refs": refs, "live": live.to(torch.int32).view(1), "pool": _bits(pool)}


def _plain_copy(s):
    s["pool"][:, s["dst"].long()] = s["pool"][:, s["src"].long()]
    return {"pool": _bits(s["pool"])}


# -- work -----------------------------------------------------------------


def work(case):
    op = case["op"]
    if op == "copy":
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": 2 * case["layers"] * case["count"] * case["H"] * case["a"] * case["b"] * size, "flops": 0}
    token = case["HKV"] * case["D"] * 2  # bytes of a token's keys, or values, in a layer
    if op == "compact":
        lens = _compact_lens(case)
        used = sum(-(-n // case["page"]) for n in lens)
        P = max(case["P"], used)
        # pages in no order: of the live ones the share (P - used) / P lies above
        moved = used * (P - used) / P
        ints = 4 * 2 * (P + case["N"] * max(-(-n // case["page"]) for n in lens))
        return {"bytes": int(2 * moved * case["page"] * token * 2 * case["layers"] + ints), "flops": 0}
    if op == "beam":
        lens, _ = _lengths(case)
        page, F = case["page"], case["F"]
        M = -(-(max(lens) + case["grow"]) // page)
        P = sum(-(-n // page) for n in lens) + F * (2 + case["grow"] // page)
        # the copied last pages; the freed and written rows of the table, the counts
        return {"bytes": F * 2 * page * token * 2 * case["layers"] + 4 * (3 * F * M + 2 * P), "flops": 0}
    lens, new = _lengths(case)
    if op == "append":
        return {"bytes": sum(new) * 2 * 2 * token, "flops": 0}
    HQ, D = case["HQ"], case["D"]
    keys = pairs = 0
    for n, t in zip(lens, new):
        w = case["window"] or n
        keys += min(n, t - 1 + w)
        # query i sees min(w, n - t + 1 + i) keys
        first = n - t + 1
        grow = max(0, min(t, w - first))
        pairs += grow * first + grow * (grow - 1) // 2 + (t - grow) * w
    nbytes = keys * 2 * token + sum(new) * HQ * D * 2 * 2 + (sum(new) * HQ * 4 if case["lse"] else 0)
    return {"bytes": nbytes, "flops": 4 * D * HQ * pairs}


# -- exact ----------------------------------------------------------------


def exact(case, seed):
    """Attention in 64 bits, sequence by sequence and head by head, from the
    definition: position p sees the keys in (p - window, p].  The other
    operators move values and count pages: nothing to be exact about."""
    if case["op"] != "attention":
        return None
    s = prepare(case, seed)
    lens, new = _lengths(case)
    page, G = case["page"], case["HQ"] // case["HKV"]
    q = s["q"].reshape(-1, case["HQ"], case["D"])
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    t0 = 0
    for n, (L, T) in enumerate(zip(lens, new)):
        pages = s["table"][n, :-(-L // page)].long()
        pos = torch.arange(L - T, L, device=q.device)[:, None]
        j = torch.arange(L, device=q.device)[None, :]
        seen = j <= pos
        if case["window"]:
            seen = seen & (j > pos - case["window"])
        for h in range(case["HKV"]):
            K = s["k"][pages, :, h].reshape(-1, case["D"])[:L].double()
            V = s["v"][pages, :, h].reshape(-1, case["D"])[:L].double()
            for g in range(h * G, (h + 1) * G):
                x = torch.mm(q[t0:t0 + T, g].double(), K.t().contiguous()) * case["D"] ** -0.5
                x = x.masked_fill(~seen, -math.inf)
                z = torch.logsumexp(x, 1, keepdim=True)
                o[t0:t0 + T, g] = torch.mm(torch.exp(x - z), V)
                lse[t0:t0 + T, g] = z[:, 0]
        t0 += T
    out = {"o": o.view(s["q"].shape)}
    if case["lse"]:
        out["lse"] = lse.view(s["q"].shape[:3])
    return out
