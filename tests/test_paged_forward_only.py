"""The paged calls have no backward: each refuses tensors that require a
gradient, where else it would be lost without a word (CPU only)."""

from __future__ import annotations

import pytest
import torch

from kda_bt16 import paged_append, paged_attention, paged_compact, paged_copy, paged_fork

BF16 = torch.bfloat16


def _i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def calls():
    """(name, a call of it with one of its tensors requiring a gradient)."""
    def grad(*shape, dtype=BF16):
        return torch.zeros(*shape, dtype=dtype, requires_grad=True)

    k, cache, table, lens = torch.zeros(2, 3, 2, 64, dtype=BF16), torch.zeros(5, 16, 2, 64, dtype=BF16), _i32(2, 4), _i32(2)
    gk, gc = grad(2, 3, 2, 64), grad(5, 16, 2, 64)
    pool, gp, rows, refs = torch.zeros(8, 16, 2, 64), grad(8, 16, 2, 64, dtype=torch.float32), _i32(2), _i32(8)
    yield "paged_attention", lambda: paged_attention(gk, cache, cache, table, lens)
    yield "paged_attention", lambda: paged_attention(k, cache, gc, table, lens)
    for args in ((gk, k, cache, cache), (k, gk, cache, cache), (gk[..., :], gk * 2, cache, cache), (k, k, gc, cache),
                 (k, k, cache, gc)):
        yield "paged_append", lambda args=args: paged_append(*args, table, lens)
    for pools in (gp, [pool, gp]):
        yield "paged_fork", lambda pools=pools: paged_fork(pools, table, lens, refs, rows, rows)
        yield "paged_copy", lambda pools=pools: paged_copy(pools, rows, rows)
        yield "paged_compact", lambda pools=pools: paged_compact(pools, table, refs)


@pytest.mark.parametrize("i", range(13))
def test_a_gradient_is_refused(i):
    name, call = list(calls())[i]
    with pytest.raises(NotImplementedError, match=f"{name} is forward only: inputs require grad"):
        call()
    # without a graph there is none to lose
    with torch.no_grad(), pytest.raises(ValueError, match="runs on a ROCm GPU"):
        call()


def test_every_call_is_tried():
    assert len(list(calls())) == 13
