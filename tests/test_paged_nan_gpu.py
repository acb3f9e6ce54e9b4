"""Queries that are not finite, over a paged cache: NaN is the answer to them,
-inf stays the log-sum-exp of queries that see no key, and the other queries'
answers are as ever."""

from __future__ import annotations

import math

import pytest
import torch

import paged_oracle as oracle
from kda_bt16 import paged_attention
from test_paged_gpu import BF16, FP16, _tol, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (FP16, 64)])
# few rows whole and cut, many rows whole and cut; the last sequence has fewer
# cached tokens than new ones, so that its first queries see no key
@pytest.mark.parametrize("T,lens", [(5, [40, 130, 3]), (5, [2000, 900, 3]), (140, [140, 200, 70]), (140, [2000, 700, 70])])
@pytest.mark.parametrize("causal", [True, False])
def test_queries_that_are_not_finite(T, lens, causal, dtype, D, gpu_device):
    dev = gpu_device
    (kc, vc), (dk, dv), table, ln, gen = make(lens, 2, D, 16, dtype, dev)
    q = torch.randn(3, T, 4, D, generator=gen).to(dtype)
    q[0, 0, 0, 3] = math.nan
    q[0, T // 2, 1] = math.nan
    q[1, T - 1, 3, 5] = math.nan
    q[1, T - 2, 0, 7] = math.inf  # scores of +inf among others: e^(inf - inf)
    q[2, 0, 2] = math.nan  # causal: sees no key
    q[2, T - 1, 2, D - 1] = math.nan
    bad = ~torch.isfinite(q).all(-1)
    want, want_lse = oracle.attention(q, kc, vc, table, ln, 0.1, causal)
    o, lse = paged_attention(q.to(dev), dk, dv, table.to(dev), ln.to(dev), scale=0.1, causal=causal, return_lse=True)
    o, lse = o.double().cpu(), lse.double().cpu()
    none = torch.isneginf(want_lse)
    assert none.any() == causal and none[2, 0, 2] == causal
    assert torch.equal(torch.isneginf(lse), none)
    assert (o[none] == 0).all()
    bad &= ~none
    assert torch.isnan(lse[bad]).all() and torch.isnan(o[bad]).all()
    fine = ~bad & ~none
    assert (o - want)[fine].abs().max() <= _tol(dtype)
    assert (lse - want_lse)[fine].abs().max() <= 1e-4
