"""The paged calls' checks of their arguments (CPU only): types and messages,
before any launch."""

from __future__ import annotations

import pytest
import torch

from kda_bt16 import (
    paged_append,
    paged_attention,
    paged_compact,
    paged_copy,
    paged_fork,
    paged_free,
    paged_reserve,
)

BF16 = torch.bfloat16


def _i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def attention(**change):
    a = dict(q=torch.zeros(2, 3, 4, 64, dtype=BF16), k_cache=torch.zeros(5, 16, 2, 64, dtype=BF16),
             v_cache=torch.zeros(5, 16, 2, 64, dtype=BF16), page_table=_i32(2, 4), seq_lens=_i32(2))
    kw = {k: change.pop(k) for k in list(change) if k not in a}
    a.update(change)
    return paged_attention(a["q"], a["k_cache"], a["v_cache"], a["page_table"], a["seq_lens"], **kw)


def test_attention_wants_a_gpu():
    with pytest.raises(ValueError, match="runs on a ROCm GPU"):
        attention()


@pytest.mark.parametrize("change,error,match", [
    (dict(q=torch.zeros(3, 4, 64, dtype=BF16)), ValueError, "q must be 4D"),
    (dict(q=torch.zeros(2, 3, 4, 64)), TypeError, "q must be torch.bfloat16 like the cache"),
    (dict(q=torch.zeros(3, 3, 4, 64, dtype=BF16)), ValueError, "one row a row of page_table, 2, got 3"),
    (dict(q=torch.zeros(2, 3, 4, 128, dtype=BF16)), ValueError, "the cache's head size 64, got 128"),
    (dict(q=torch.zeros(2, 3, 3, 64, dtype=BF16)), ValueError, "HQ must be a multiple of HKV"),
    (dict(q=torch.zeros(2, 0, 4, 64, dtype=BF16)), ValueError, "q dimensions must be positive"),
    (dict(q=torch.zeros(2, 3, 64, 4, dtype=BF16).transpose(2, 3)), ValueError, "q's last dimension must be contiguous"),
    (dict(q=torch.zeros(2, 3, 4, 68, dtype=BF16)[..., :64]), ValueError, "strides multiples of 8"),
    (dict(q=torch.zeros(2, 3, 4, 64, dtype=BF16, requires_grad=True)), NotImplementedError, "forward only"),
    (dict(k_cache=torch.zeros(5, 16, 64, dtype=BF16)), ValueError, "k_cache must be 4D"),
    (dict(k_cache=torch.zeros(5, 16, 2, 64)), TypeError, "k_cache must be bfloat16 or float16"),
    (dict(v_cache=torch.zeros(5, 16, 2, 64, dtype=torch.float16)), TypeError, "v_cache must be torch.bfloat16"),
    (dict(v_cache=torch.zeros(5, 32, 2, 64, dtype=BF16)), ValueError, "v_cache.shape"),
    (dict(k_cache=torch.zeros(5, 24, 2, 64, dtype=BF16), v_cache=torch.zeros(5, 24, 2, 64, dtype=BF16)), ValueError,
     "power of two from 16 to 1024, got 24"),
    (dict(k_cache=torch.zeros(5, 8, 2, 64, dtype=BF16), v_cache=torch.zeros(5, 8, 2, 64, dtype=BF16)), ValueError,
     "power of two"),
    (dict(k_cache=torch.zeros(5, 16, 2, 96, dtype=BF16), v_cache=torch.zeros(5, 16, 2, 96, dtype=BF16)), ValueError,
     "head size must be 64 or 128"),
    (dict(k_cache=torch.zeros(5, 1, 2, 64, dtype=BF16).expand(5, 16, 2, 64)), ValueError, "tokens must not overlap"),
    (dict(k_cache=torch.zeros(0, 16, 2, 64, dtype=BF16), v_cache=torch.zeros(0, 16, 2, 64, dtype=BF16)), ValueError,
     "cache dimensions must be positive"),
    (dict(page_table=torch.zeros(2, 4, dtype=torch.int64)), TypeError, "page_table must be int32"),
    (dict(page_table=_i32(8)), ValueError, "page_table must be 2D"),
    (dict(page_table=_i32(2, 0)), ValueError, "page_table dimensions must be positive"),
    (dict(page_table=_i32(1, 4).expand(2, 4)), ValueError, "rows of page_table must not overlap"),
    (dict(page_table=_i32(4, 2).t()), ValueError, "page_table must be contiguous"),
    (dict(seq_lens=_i32(3)), ValueError, "seq_lens must have one entry a row"),
    (dict(seq_lens=torch.zeros(2)), TypeError, "seq_lens must be int32"),
    (dict(scale=0.0), ValueError, "scale must be positive"),
    (dict(scale=-1.0), ValueError, "scale must be positive"),
    (dict(scale=float("nan")), ValueError, "scale must be positive"),
    (dict(window=0), ValueError, "window must be at least 1"),
    (dict(window=5, causal=False), ValueError, "window needs causal=True"),
    (dict(cu_seqlens=_i32(3)), ValueError, "batch size is expected to be 1"),
    (dict(q=torch.zeros(1, 6, 4, 64, dtype=BF16), cu_seqlens=_i32(2)), ValueError, "cu_seqlens must have 3 entries"),
    (dict(q=torch.zeros(1, 6, 4, 64, dtype=BF16), cu_seqlens=torch.zeros(3)), TypeError, "cu_seqlens must be int32 or"),
    (dict(q=torch.zeros(1, 6, 4, 64, dtype=BF16), cu_seqlens=_i32(6)[::2]), ValueError, "cu_seqlens must be contiguous"),
])
def test_attention_refuses(change, error, match):
    with pytest.raises(error, match=match):
        attention(**change)


@pytest.mark.parametrize("change,error,match", [
    (dict(k=torch.zeros(2, 3, 4, 64, dtype=BF16)), ValueError, "k must have the cache's 2 heads, got 4"),
    (dict(v=torch.zeros(2, 4, 2, 64, dtype=BF16)), ValueError, "v.shape"),
    (dict(v=torch.zeros(2, 3, 2, 64)), TypeError, "v must be torch.bfloat16"),
    (dict(), ValueError, "runs on a ROCm GPU"),
])
def test_append_refuses(change, error, match):
    a = dict(k=torch.zeros(2, 3, 2, 64, dtype=BF16), v=torch.zeros(2, 3, 2, 64, dtype=BF16)) | change
    cache = torch.zeros(5, 16, 2, 64, dtype=BF16)
    with pytest.raises(error, match=match):
        paged_append(a["k"], a["v"], cache, cache.clone(), _i32(2, 4), _i32(2))


def test_page_calls_refuse():
    table, lens, refs, pool = _i32(3, 4), _i32(3), _i32(8), torch.zeros(2, 8, 16, 2, 64)
    rows = _i32(2)
    with pytest.raises(ValueError, match="new_tokens must have 3 entries"):
        paged_reserve(table, lens, refs, rows, 16)
    with pytest.raises(ValueError, match="power of two"):
        paged_reserve(table, lens, refs, lens.clone(), 20)
    with pytest.raises(TypeError, match="new_tokens must be int32"):
        paged_reserve(table, lens, refs, lens.long(), 16)
    with pytest.raises(TypeError, match="page_refs must be int32"):
        paged_free(table, lens, refs.long(), rows)
    with pytest.raises(ValueError, match="page_refs must not be empty"):
        paged_free(table, lens, _i32(0), rows)
    with pytest.raises(ValueError, match="page_refs must be 16-byte aligned"):
        paged_free(table, lens, _i32(9)[1:], rows)
    with pytest.raises(TypeError, match="rows must be int32"):
        paged_free(table, lens, refs, rows.long())
    with pytest.raises(ValueError, match="src must be 1D"):
        paged_fork(pool, table, lens, refs, _i32(2, 1), rows)
    with pytest.raises(ValueError, match="dst must have 2 entries"):
        paged_fork(pool, table, lens, refs, rows, _i32(3))
    with pytest.raises(ValueError, match="page_refs must have one entry a page, 8, got 9"):
        paged_fork(pool, table, lens, _i32(9), rows, rows)
    with pytest.raises(ValueError, match="power of two"):
        paged_fork(torch.zeros(8, 2, 16, 64), table, lens, refs, rows, rows)  # page_size not third from the end
    with pytest.raises(ValueError, match="must be contiguous"):
        paged_copy(pool.transpose(0, 1), rows, rows)
    with pytest.raises(ValueError, match="at least 4D"):
        paged_copy(torch.zeros(8, 16, 2), rows, rows)
    with pytest.raises(ValueError, match="pages multiples of 16 bytes"):
        paged_copy(torch.zeros(8, 1, 1, 3), rows, rows)
    with pytest.raises(ValueError, match="dimensions must be positive"):
        paged_copy(torch.zeros(8, 0, 1, 4), rows, rows)
    with pytest.raises(ValueError, match="pool 1 must have 8 pages like the first, got 9"):
        paged_copy([pool, torch.zeros(9, 16, 2, 64)], rows, rows)
    with pytest.raises(ValueError, match="between 1 and 8 pools, got 0"):
        paged_copy([], rows, rows)
    with pytest.raises(ValueError, match="between 1 and 8 pools, got 9"):
        paged_copy([pool] * 9, rows, rows)
    with pytest.raises(ValueError, match="page_refs must have one entry a page"):
        paged_compact(pool, table, _i32(12))
    with pytest.raises(TypeError, match="page_table must be int32"):
        paged_compact(pool, table.long(), refs)
    for call in (lambda: paged_reserve(table, lens, refs, lens.clone(), 16), lambda: paged_free(table, lens, refs, rows),
                 lambda: paged_fork(pool, table, lens, refs, rows, rows), lambda: paged_copy(pool, rows, rows),
                 lambda: paged_compact(pool, table, refs)):
        with pytest.raises(ValueError, match="runs on a ROCm GPU"):
            call()
