"""How far paged_attention's outputs may be from 64 bits, following their size.

With U the largest relative error of one rounding to the cache's type (2^-8 for
bf16, 2^-11 for fp16), w the softmax's weights and v the values:

* every exponential is rounded once, o once: U * sum(w |v|) + U |o|;
* fp16 exponentials below 2^-14 of the running maximum's are subnormal, off by
  2^-25 at most, over a sum of at least 1: 2^-25 * L * mean |v|, below 2^-25 * L;
* fp32: a score of D products is off by at most D * 2^-24 * scale * |q| |k|, with
  entries of unit variance |q| |k| below 1.3 * D; sums of L terms by L * 2^-24 of
  their size, one each above and below the fraction; 64 * 2^-24 for the rest.

So much for a single element.  Over a sequence the errors are independent of
one another: a rounding's root mean square is at most U / sqrt(3), and values
of mean 0 make o's as large as that of its terms.  Relative to o's the error's
root mean square is then at most U * sqrt(2 / 3): 0.0032 and 0.0004, taken as
0.004 and 0.0005 for samples of at least 64 numbers.
"""

from __future__ import annotations

import math

import torch

import paged_oracle as oracle

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
RMS = {torch.bfloat16: 0.004, torch.float16: 0.0005}


def expected(q, k_cache, v_cache, table, lens, scale, causal=True, window=None, cu=None):
    """(o, lse, sum of w |v|), in 64 bits."""
    o, lse = oracle.attention(q, k_cache, v_cache, table, lens, scale, causal, window, cu)
    return o, lse, oracle.attention(q, k_cache, v_cache.abs(), table, lens, scale, causal, window, cu)[0]


def misses(o, lse, want, q, lens, scale, cu=None):
    """What is out of bounds, as a list of texts (``want``: expected()'s)."""
    exact, exact_lse, mass = want
    D, u, out = q.shape[-1], U[q.dtype], []
    o, lse = o.double().cpu(), lse.double().cpu()
    none = torch.isneginf(exact_lse)
    if not torch.equal(torch.isneginf(lse), none) or bool((o[none] != 0).any()) or not bool(torch.isfinite(o).all()):
        return ["queries that see no key"]
    for n, (first, count) in enumerate(oracle.spans(len(lens), q.shape[1], cu)):
        L = int(lens[n])
        if count == 0 or L == 0:
            continue
        got, x, m = (t.reshape(-1, *t.shape[2:])[first:first + count] for t in (o, exact, mass))
        z, e = (t.reshape(-1, t.shape[2])[first:first + count] for t in (lse, exact_lse))
        fp32 = 2.0 ** -24 * (2 * D * scale * 1.3 * D + 2 * L + 64)
        limit = (u + fp32) * m + u * x.abs() + (2.0 ** -25 * L if q.dtype == torch.float16 else 0) + 1e-7
        over = ((got - x).abs() / limit).max().item()
        if over > 1:
            out.append(f"sequence {n}: an element of o by {over:.2f} of its bound")
        some = ~torch.isneginf(e)
        rms = ((got - x)[some].pow(2).mean() / x[some].pow(2).mean()).sqrt().item() if some.any() else 0.0
        if rms > RMS[q.dtype]:
            out.append(f"sequence {n}: root mean square {rms:.5f}")
        far = (z - e)[some].abs().max().item() if some.any() else 0.0
        if far > fp32:
            out.append(f"sequence {n}: lse by {far}")
    return out


def rounded(q, k_cache, v_cache, table, lens, scale):
    """o as rounding the exponentials and the result once gives it, else in 64
    bits (causal, one batch row a sequence)."""
    N, T, HQ, D = q.shape
    G = HQ // k_cache.shape[2]
    o = torch.zeros(q.shape, dtype=q.dtype)
    for n in range(N):
        L = int(lens[n])
        hide = torch.arange(L) > torch.arange(L - T, L)[:, None]
        for h in range(HQ):
            K, V = (oracle.cached(c, table, n, L, h // G) for c in (k_cache, v_cache))
            x = (scale * (q[n, :, h].double() @ K.t())).masked_fill(hide, -math.inf)
            e = torch.exp(x - x.amax(1, keepdim=True))
            o[n, :, h] = (e.to(q.dtype).double() @ V / e.sum(1, keepdim=True)).to(q.dtype)
    return o
