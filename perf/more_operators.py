"""Three operators next to the paged cache's, as cases to time and to compare.

A cache is a pool of pages of ``page`` tokens, ``[P, page, HKV, D]`` for the
keys and for the values of a layer.  ``page_table [N, M]`` names the pages
of each sequence (-1: none), ``seq_lens [N]`` counts its cached tokens (new
ones included).  New tokens are ``[N, T, heads, D]``, or packed ``[1, total,
heads, D]`` with the offsets ``cu_seqlens``.

A case is a dict of plain values.  ``op`` is

* ``rotary``: new queries and keys turned by their positions, the keys and
  values into their places in the pages on the way;
* ``sinks``: attention over a sliding window and a few first tokens that stay
  visible;
* ``shared``: attention of sequences in groups that share their first tokens,
  which are looked at once for the whole group.

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


def _rotary(name, N, T, lo, hi, HQ, HKV, D=128, rotary=0, interleaved=False, base=10000.0, page=16, dtype="bf16",
            packed=False, layout="token", spread=1):
    return {"name": name, "op": "rotary", "N": N, "T": T, "lo": lo, "hi": hi, "HQ": HQ, "HKV": HKV, "D": D,
            "rotary": rotary or D, "interleaved": interleaved, "base": base, "page": page, "dtype": dtype,
            "packed": packed, "layout": layout, "spread": spread}


def _sinks(name, N, T, lo, hi, HQ, HKV, window, sinks, D=128, page=16, dtype="bf16", packed=False, lse=False,
           layout="token", spread=1):
    return {"name": name, "op": "sinks", "N": N, "T": T, "lo": lo, "hi": hi, "HQ": HQ, "HKV": HKV, "window": window,
            "sinks": sinks, "D": D, "page": page, "dtype": dtype, "packed": packed, "lse": lse, "layout": layout,
            "spread": spread}


def _shared(name, groups, few, most, plo, phi, T, lo, hi, HQ, HKV, D=128, page=16, dtype="bf16", packed=False, lse=False,
            layout="token", spread=1):
    """``groups`` groups of ``few`` to ``most`` sequences; ``plo`` to ``phi``
    shared tokens, ``lo`` to ``hi`` tokens of a sequence's own behind them."""
    return {"name": name, "op": "shared", "groups": groups, "few": few, "most": most, "plo": plo, "phi": phi, "T": T,
            "lo": lo, "hi": hi, "HQ": HQ, "HKV": HKV, "D": D, "page": page, "dtype": dtype, "packed": packed,
            "lse": lse, "layout": layout, "spread": spread}


def listed():
    return [
        # The next token of one long conversation: the smallest call, where
        # latency counts.
        _rotary("rotary_1x1", 1, 1, 20000, 20000, 32, 8, base=500000.0),
        # The next token of each of 128 conversations.
        _rotary("rotary_128x1", 128, 1, 100, 2000, 32, 8, layout="head"),
        # 16 prompts of uneven lengths, packed; fp16, small heads in groups of
        # 6, half of each turned, in neighbouring pairs.
        _rotary("rotary_packed16_fp16_d64", 16, 1024, 1024, 6000, 24, 4, D=64, rotary=32, interleaved=True, page=32,
                dtype="fp16", packed=True),
        # One long prompt.
        _rotary("rotary_1x8192", 1, 8192, 8192, 8192, 32, 8),
        # A decode step of one conversation far beyond its window.
        _sinks("sinks_1x8000", 1, 1, 8000, 8000, 32, 8, 1024, 4),
        # A decode step of a full serving batch, some conversations shorter
        # than the window, most beyond it.
        _sinks("sinks_64_ragged", 64, 1, 100, 16000, 32, 8, 4096, 4, layout="head"),
        # A packed batch of a serving step: chunks and single tokens; a number
        # of first tokens that ends inside a page; fp16, small heads; with the
        # log-sum-exp.
        _sinks("sinks_packed8_fp16_d64", 8, 1024, 900, 12000, 24, 4, 1000, 70, D=64, page=64, dtype="fp16", packed=True,
               lse=True),
        # One long prompt under a window.
        _sinks("sinks_1x8192", 1, 8192, 8192, 8192, 32, 8, 2048, 64),
        # The beams of one short prompt, a decode step.
        _shared("shared_beam8", 1, 8, 8, 2000, 2000, 1, 1, 60, 32, 8),
        # 64 answers sampled from one long prompt, a decode step.
        _shared("shared_64_of_16000", 1, 64, 64, 16000, 16000, 1, 10, 500, 32, 8, layout="head"),
        # Drafts of 5 tokens in 6 groups behind prompts of uneven lengths (a
        # system prompt each); fp16, small heads in groups of 6; with the
        # log-sum-exp.
        _shared("shared_draft_6x12_fp16_d64", 6, 3, 12, 300, 8000, 5, 5, 700, 24, 4, D=64, page=32, dtype="fp16", lse=True),
        # 8 questions about one long document, packed: the largest.
        _shared("shared_chunk_8_of_12000", 1, 8, 8, 12000, 12000, 512, 512, 600, 32, 8, page=64, packed=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _unnamed(case):
    return {k: v for k, v in case.items() if k != "name"}


def draw(rng):
    op = rng.choice(["rotary", "sinks", "shared"])
    kind = rng.choice(["decode", "draft", "chunk", "chunk"])
    HKV = rng.choice([1, 2, 4, 8])
    HQ = min(32, HKV * rng.choice([1, 2, 4, 6, 8]))
    HQ -= HQ % HKV
    D = rng.choice([64, 128, 128])
    kw = {"D": D, "page": rng.choice([16, 16, 32, 64, 128]), "dtype": rng.choice(["bf16", "bf16", "fp16"]),
          "layout": rng.choice(["token", "head"]), "spread": rng.randrange(1, 1 << 20)}
    if op == "rotary":
        N, T = _log_int(rng, 1, 128), 1 if kind == "decode" else _log_int(rng, 2, 8192)
        T = max(1, min(T, 8192 // N))
        lo = _log_int(rng, max(T, 50), 8192)
        hi = _log_int(rng, lo, max(lo, min(32000, 128 * 2000 // N)))
        return _unnamed(_rotary("", N, T, lo, hi, HQ, HKV, rotary=rng.choice([D, D, D // 2, D // 4, 3 * D // 4]),
                                interleaved=rng.random() < 0.4, base=rng.choice([10000.0, 500000.0]),
                                packed=T > 1 and rng.random() < 0.6, **kw))
    kw["lse"] = rng.random() < 0.3
    kw["packed"] = kind == "chunk" and rng.random() < 0.7
    T = {"decode": 1, "draft": rng.randint(2, 8), "chunk": _log_int(rng, 9, 1024)}[kind]
    if op == "sinks":
        window, sinks = _log_int(rng, 16, 4096), _log_int(rng, 1, 256)
        if kind == "chunk":
            N = rng.randint(1, 8)
            if rng.random() < 0.3:
                N, T = 1, _log_int(rng, 1000, 8192)
        else:
            N = _log_int(rng, 1, 128)
        lo = _log_int(rng, max(T, 20), max(T, 4000))
        # the products, and the keys
        window = max(16, min(window, 8192 * 1800 * 32 * 128 // (N * T * HQ * D) - sinks, 64 * 1800 * 8 * 128 // (N * HKV * D)))
        # the scores of the plain form, and the keys it gathers
        most = min(8192 * 8192 * 32 // (N * T * HQ), 64 * 16000 // N, 32000)
        return _unnamed(_sinks("", N, T, lo, max(lo, min(_log_int(rng, lo, max(lo, 32000)), most)), HQ, HKV, window, sinks,
                               **kw))
    groups = _log_int(rng, 1, 16)
    most = _log_int(rng, 1, max(1, 128 // groups))
    if kind == "chunk":
        groups, most, T = min(groups, 4), min(most, 4), min(T, 512)
    few = rng.randint(1, most)
    lo = rng.randint(T, T + 20)
    hi = _log_int(rng, lo, lo + 1000)
    plo = _log_int(rng, 16, 4000)
    N = groups * most
    # the keys that the plain form gathers, and the products
    top = min(64 * 16000 // N, 8192 * 1800 * 32 * 128 // (N * T * HQ * D)) - hi
    plo = max(16, min(plo, top))
    phi = max(plo, min(_log_int(rng, plo, 16000), top))
    return _unnamed(_shared("", groups, few, most, plo, phi, T, lo, hi, HQ, HKV, **kw))


# -- lengths and tables ---------------------------------------------------


def _members(case):
    """(shared tokens, sequences) of each group of a ``shared`` case."""
    rng = random.Random(case["spread"] + 1)
    return [(_log_int(rng, case["plo"], case["phi"]), rng.randint(case["few"], case["most"])) for _ in
            range(case["groups"])]


def _lengths(case):
    """(cached tokens, new tokens) of each sequence: the cached ones spread by
    their logarithm between lo and hi (``shared``: those of its own, behind
    the group's), in packed batches the new ones from a single token up to T
    (the last sequence's T)."""
    rng = random.Random(case["spread"])
    before = [0] * case.get("N", 0)
    if case["op"] == "shared":
        before = [shared for shared, count in _members(case) for _ in range(count)]
    lens = [x + _log_int(rng, case["lo"], case["hi"]) for x in before]
    T = case["T"]
    new = [T] * len(lens)
    if case["packed"]:
        new = [1 if rng.random() < 0.35 else _log_int(rng, 1, T) for _ in lens[:-1]] + [T]
    return lens, new


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _table(lens, page, gen):
    """A page table of pages in no order, and the number of pages of its pool."""
    need = [-(-n // page) for n in lens]
    P = sum(need) + 3
    order = torch.randperm(P, generator=gen, device="cuda", dtype=torch.int32)
    at = torch.tensor(need, device="cuda")
    start = torch.cumsum(at, 0) - at
    col = torch.arange(max(need), device="cuda")
    idx = (start[:, None] + col).clamp_(max=P - 1)
    return torch.where(col < at[:, None], order[idx], torch.full_like(idx, -1, dtype=torch.int32)).contiguous(), P


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
    return _int32([0] + new).cumsum(0, dtype=torch.int32)


# -- prepare --------------------------------------------------------------


def prepare(case, seed):
    gen = _gen(seed)
    lens, new = _lengths(case)
    table, P = _table(lens, case["page"], gen)
    s = {"case": case}
    if case["op"] == "shared":
        table, s["groups"], s["shared"] = _share(case, table)
    s["k"], s["v"] = _cache(case, P, gen)
    if case["op"] == "shared":
        _same_last_page(case, s["k"], s["v"], table)
    s |= {"table": table, "lens": _int32(lens), "cu": _cu(new) if case["packed"] else None, "tmax": max(new)}
    dt, HQ, HKV, D = _DTYPES[case["dtype"]], case["HQ"], case["HKV"], case["D"]
    shape = (1, sum(new)) if case["packed"] else (len(lens), case["T"])
    if case["op"] == "rotary":
        # as a fused projection leaves them, side by side
        s["qkv"] = _randn(gen, dt, *shape, HQ + 2 * HKV, D)
        half = case["rotary"] // 2
        s["freq"] = (case["base"] ** (-torch.arange(half, dtype=torch.float64) / half)).float().cuda()
    else:
        s["q"] = _randn(gen, dt, *shape, HQ, D)
        s["scale"] = D ** -0.5
    return s


def _share(case, table):
    """Every sequence of a group gets the first one's whole pages of the shared
    tokens: what forking leaves.  The groups' offsets and shared tokens."""
    n, offsets, shared = 0, [0], []
    for tokens, count in _members(case):
        whole = tokens // case["page"]
        table[n:n + count, :whole] = table[n, :whole].clone()
        n += count
        offsets.append(n)
        shared.append(tokens)
    return table, _int32(offsets), _int32(shared)


def _same_last_page(case, k, v, table):
    """The shared tokens of a partial page, a page of every sequence's own
    with the same contents."""
    n = 0
    for tokens, count in _members(case):
        if tokens % case["page"] and count > 1:
            pages = table[n:n + count, tokens // case["page"]].long()
            k[pages[1:]] = k[pages[0]].clone()
            v[pages[1:]] = v[pages[0]].clone()
        n += count


# -- run ------------------------------------------------------------------


def _bits(t):
    """A tensor's values as whole numbers, for what is only moved."""
    return t.view(torch.int16)


def run(state):
    op = state["case"]["op"]
    if own:
        return {"rotary": _own_rotary, "sinks": _own_sinks, "shared": _own_shared}[op](state)
    return {"rotary": _plain_rotary, "sinks": _plain_attention, "shared": _plain_attention}[op](state)


def _package():
    path = os.path.join(os.getcwd(), "kda-ascendc_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import kda_bt16

    return kda_bt16


def _split(s):
    HQ, HKV = s["case"]["HQ"], s["case"]["HKV"]
    return s["qkv"].split([HQ, HKV, HKV], 2)


def _own_rotary(s):
    q, k, v = _split(s)
    q = _package().paged_append_rotary(q, k, v, s["k"], s["v"], s["table"], s["lens"], s["freq"],
                                       interleaved=s["case"]["interleaved"], cu_seqlens=s["cu"])
    return {"q": q, "k": s["k"], "v": _bits(s["v"])}


def _own_sinks(s):
    lse = s["case"]["lse"]
    r = _package().paged_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], scale=s["scale"],
                                   window=s["case"]["window"], sinks=s["case"]["sinks"], cu_seqlens=s["cu"], return_lse=lse)
    return {"o": r[0], "lse": r[1]} if lse else {"o": r}


def _own_shared(s):
    lse = s["case"]["lse"]
    r = _package().paged_attention_shared(s["q"], s["k"], s["v"], s["table"], s["lens"], s["groups"], s["shared"],
                                          scale=s["scale"], cu_seqlens=s["cu"], return_lse=lse)
    return {"o": r[0], "lse": r[1]} if lse else {"o": r}


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


def _turn(x, cos, sin, interleaved):
    """x [tokens, heads, D] in 32 bits, the first 2 * len(cos) elements turned
    in pairs: neighbours, or element i and i + len(cos)."""
    half = cos.shape[-1]
    cos, sin = cos[:, None], sin[:, None]
    turned = x[..., :2 * half]
    a, b = (turned[..., ::2], turned[..., 1::2]) if interleaved else (turned[..., :half], turned[..., half:])
    a, b = a * cos - b * sin, b * cos + a * sin
    both = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([both, x[..., 2 * half:]], -1)


def _plain_rotary(s):
    q, k, v = _split(s)
    tokens = q.shape[0] * q.shape[1]
    n, pos = _places(s, tokens)
    angle = pos.double()[:, None] * s["freq"].double()  # (a far position's turns leave 32 bits nothing behind the point)
    cos, sin = angle.cos().float(), angle.sin().float()
    turn = [_turn(x.reshape(tokens, *x.shape[2:]).float(), cos, sin, s["case"]["interleaved"]).to(x.dtype) for x in (q, k)]
    page = s["k"].shape[1]
    at = s["table"].long()[n, pos // page]
    s["k"][at, pos % page] = turn[1]
    s["v"][at, pos % page] = v.reshape(tokens, *v.shape[2:])
    return {"q": turn[0].view(q.shape), "k": s["k"], "v": _bits(s["v"])}


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
    if s["case"]["op"] == "sinks":
        hide |= (j <= at - s["case"]["window"]) & (j >= s["case"]["sinks"])
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


# -- work -----------------------------------------------------------------


def work(case):
    lens, new = _lengths(case)
    HQ, HKV, D = case["HQ"], case["HKV"], case["D"]
    if case["op"] == "rotary":
        # queries, keys and values in and out; 6 operations a pair
        turned = sum(new) * (HQ + HKV) * case["rotary"] // 2
        return {"bytes": sum(new) * (HQ + 2 * HKV) * D * 2 * 2 + case["rotary"] * 2, "flops": 6 * turned}
    keys = pairs = 0
    for n, t in zip(lens, new):
        if case["op"] == "shared":
            pairs += t * (n - t) + t * (t + 1) // 2
            keys += n
            continue
        w, s = case["window"], case["sinks"]
        # the first tokens, and the window of the first new token up to the end
        start = max(0, n - t + 1 - w)
        keys += n - max(0, start - s)
        for p in range(n - t, n):
            pairs += p + 1 - max(0, max(0, p + 1 - w) - s)
    if case["op"] == "shared":
        keys -= sum(shared * (count - 1) for shared, count in _members(case))
    nbytes = keys * 2 * 2 * HKV * D + sum(new) * HQ * D * 2 * 2 + (sum(new) * HQ * 4 if case["lse"] else 0)
    return {"bytes": nbytes, "flops": 4 * D * HQ * pairs}


# -- exact ----------------------------------------------------------------


def exact(case, seed):
    """In 64 bits, sequence by sequence, from the definitions."""
    s = prepare(case, seed)
    lens, new = _lengths(case)
    return _exact_rotary(s, lens, new) if case["op"] == "rotary" else _exact_attention(s, lens, new)


def _exact_rotary(s, lens, new):
    """A pair (a, b) is a number a + bi, turned by e^(i * position * frequency)."""
    case, page = s["case"], s["case"]["page"]
    freq, half = s["freq"].double(), s["case"]["rotary"] // 2
    i = torch.arange(half, device=freq.device)
    first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
    x = s["qkv"].reshape(-1, *s["qkv"].shape[2:]).double()
    out_k = s["k"].double()
    t0 = 0
    for n, (L, T) in enumerate(zip(lens, new)):
        pos = torch.arange(L - T, L, device=freq.device)
        by = torch.polar(torch.ones(T, half, dtype=torch.float64, device=freq.device), pos[:, None] * freq)
        mine = x[t0:t0 + T, :case["HQ"] + case["HKV"]]
        z = torch.complex(mine[..., first], mine[..., second]) * by[:, None]
        mine[..., first], mine[..., second] = z.real, z.imag
        out_k[s["table"][n].long()[pos // page], pos % page] = mine[:, case["HQ"]:]
        t0 += T
    q = x[:, :case["HQ"]].reshape(*s["qkv"].shape[:2], case["HQ"], case["D"])
    return {"q": q, "k": out_k, "v": None}


def _exact_attention(s, lens, new):
    case = s["case"]
    page, D, G = case["page"], case["D"], case["HQ"] // case["HKV"]
    q = s["q"].reshape(-1, case["HKV"], G, D)
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.zeros(q.shape[:3], dtype=torch.float64, device=q.device)
    t0 = 0
    for n, (L, T) in enumerate(zip(lens, new)):
        pages = s["table"][n, :-(-L // page)].long()
        pos = torch.arange(L - T, L, device=q.device)[:, None]
        j = torch.arange(L, device=q.device)[None, :]
        seen = j <= pos
        if case["op"] == "sinks":
            seen = seen & ((j > pos - case["window"]) | (j < case["sinks"]))
        seen = seen.repeat_interleave(G, 0)
        for h in range(case["HKV"]):
            K = s["k"][pages, :, h].reshape(-1, D)[:L].double()
            V = s["v"][pages, :, h].reshape(-1, D)[:L].double()
            x = torch.mm(q[t0:t0 + T, h].reshape(T * G, D).double(), K.t().contiguous()) * D ** -0.5
            x = x.masked_fill_(~seen, -math.inf)
            z = torch.logsumexp(x, 1, keepdim=True)
            o[t0:t0 + T, h] = torch.mm(x.sub_(z).exp_(), V).view(T, G, D)
            lse[t0:t0 + T, h] = z.view(T, G)
        t0 += T
    out = {"o": o.view(s["q"].shape)}
    if case["lse"]:
        out["lse"] = lse.view(s["q"].shape[:3])
    return out
