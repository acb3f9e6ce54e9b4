"""A paged cache of keys and values on MI355X: attention of new tokens over
it, their append, and the work on its pages.

For models that alternate KDA layers with softmax-attention layers: the KDA
layers keep a state of fixed size (:func:`kda_bt16.kda_decode_step`), the
attention layers a cache that grows with every token.  No counterpart in the
reference, which has no attention cache.

The cache of a layer is a pool of pages for its keys and one for its values,
``[P, page_size, HKV, D]`` each: views of any layout whose last dimension is
contiguous (tokens of a head together, ``[P, HKV, page_size, D]`` transposed,
read in longer pieces).  One table serves all layers:

* ``page_table`` ``[N, M]`` int32: the pages of each sequence, from the first
  entry on, -1 for none;
* ``seq_lens`` ``[N]`` int32: its cached tokens, those of the call included;
* ``page_refs`` ``[P]`` int32: the sequences that hold each page, 0 if it is
  free.

All of it stays on the device: no call here waits for the GPU or reads a
length on the host.  A step of a serving loop::

    ok = paged_reserve(page_table, seq_lens, page_refs, new_tokens, page_size)
    for layer in layers:
        paged_append(k, v, layer.k_cache, layer.v_cache, page_table, seq_lens)
        o = paged_attention(q, layer.k_cache, layer.v_cache, page_table, seq_lens)

The new tokens of a sequence are its last ones: token i of T sits at position
``seq_lens - T + i``.  Lowering ``seq_lens`` takes a sequence's last tokens
back, those of a rejected draft; the pages behind its new length stay its own
until it grows into them (:func:`paged_reserve`) or ends.  It must not become
shorter than what it shares with a fork: its next tokens go into the page that
it then ends in.

Entries outside ``[0, P)``, lengths beyond the table's rows and row numbers
outside ``[0, N)`` give unspecified results but never an access outside the
tensors.  Forward only: where gradients are recorded, keys,
values, queries, caches and pools that require one are refused.
"""

from __future__ import annotations

import torch

from . import _hip, workspace
from .kernels import _raw_stream, _require_gpu

_CU_DTYPES = {torch.int32: _hip.DTYPE_I32, torch.int64: _hip.DTYPE_I64}
_CACHE_DTYPES = {torch.bfloat16: _hip.PAGED_BF16, torch.float16: _hip.PAGED_FP16}


def _int32(name: str, t: torch.Tensor, ndim: int, device: torch.device) -> None:
    if t.ndim != ndim:
        raise ValueError(f"{name} must be {ndim}D, got {t.ndim}D with shape {tuple(t.shape)}")
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32, got {t.dtype}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name} must be contiguous")
    if t.device != device:
        raise ValueError(f"{name} device {t.device} must match ({device})")


def _check_table(page_table, seq_lens, device) -> None:
    _int32("page_table", page_table, 2, device)
    _int32("seq_lens", seq_lens, 1, device)
    if page_table.shape[0] < 1 or page_table.shape[1] < 1:
        raise ValueError(f"page_table dimensions must be positive, got shape {tuple(page_table.shape)}")
    if seq_lens.shape[0] != page_table.shape[0]:
        raise ValueError(
            f"seq_lens must have one entry a row of page_table, {page_table.shape[0]}, got {seq_lens.shape[0]}")
    if page_table.shape[0] > 1 and page_table.stride(0) < page_table.shape[1]:
        raise ValueError("rows of page_table must not overlap")


def _check_page_size(size: int) -> None:
    if size < 16 or size > 1024 or size & (size - 1):
        raise ValueError(f"the page size must be a power of two from 16 to 1024, got {size}")


def _check_strided(name: str, t: torch.Tensor) -> None:
    """16-byte accesses at any (page, token, head)."""
    if t.stride(-1) != 1:
        raise ValueError(f"{name}'s last dimension must be contiguous")
    if t.data_ptr() % 16 or any(t.stride(i) % 8 for i in range(t.ndim - 1) if t.shape[i] > 1):
        raise ValueError(f"{name} must be 16-byte aligned, its strides multiples of 8 elements; "
                         f"got strides {t.stride()}")


def _check_cache(k_cache, v_cache, page_table, seq_lens) -> None:
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if t.ndim != 4:
            raise ValueError(f"{name} must be 4D [P, page_size, HKV, D], got {t.ndim}D with shape {tuple(t.shape)}")
        if t.dtype not in _CACHE_DTYPES:
            raise TypeError(f"{name} must be bfloat16 or float16, got {t.dtype}")
    if v_cache.shape != k_cache.shape:
        raise ValueError(f"v_cache.shape {tuple(v_cache.shape)} must match k_cache {tuple(k_cache.shape)}")
    if v_cache.dtype != k_cache.dtype:
        raise TypeError(f"v_cache must be {k_cache.dtype} like k_cache, got {v_cache.dtype}")
    P, size, HKV, D = k_cache.shape
    if P < 1 or HKV < 1:
        raise ValueError(f"cache dimensions must be positive, got P={P}, HKV={HKV}")
    _check_page_size(size)
    if D not in (64, 128):
        raise ValueError(f"the head size must be 64 or 128, got {D}")
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        _check_strided(name, t)
        if t.stride(1) < D or (P > 1 and t.stride(0) < 1) or (HKV > 1 and t.stride(2) < D):
            raise ValueError(f"{name}'s tokens must not overlap, got strides {t.stride()}")
    if v_cache.device != k_cache.device:
        raise ValueError(f"v_cache device {v_cache.device} must match k_cache ({k_cache.device})")
    _check_table(page_table, seq_lens, k_cache.device)


def _check_new(name: str, t: torch.Tensor, heads: int | None, k_cache, page_table, cu_seqlens) -> None:
    """Tensors of the new tokens: [N, T, heads, D], or [1, T, heads, D] packed."""
    if t.ndim != 4:
        raise ValueError(f"{name} must be 4D [B, T, H, D], got {t.ndim}D with shape {tuple(t.shape)}")
    if t.dtype != k_cache.dtype:
        raise TypeError(f"{name} must be {k_cache.dtype} like the cache, got {t.dtype}")
    if t.device != k_cache.device:
        raise ValueError(f"{name} device {t.device} must match k_cache ({k_cache.device})")
    B, T, H, D = t.shape
    if D != k_cache.shape[-1]:
        raise ValueError(f"{name} must have the cache's head size {k_cache.shape[-1]}, got {D}")
    if heads is not None and H != heads:
        raise ValueError(f"{name} must have the cache's {heads} heads, got {H}")
    if T < 1 or H < 1:
        raise ValueError(f"{name} dimensions must be positive, got T={T}, H={H}")
    N = page_table.shape[0]
    if cu_seqlens is None:
        if B != N:
            raise ValueError(f"{name} must have one row a row of page_table, {N}, got {B}")
    else:
        if B != 1:
            raise ValueError(
                f"The batch size is expected to be 1 rather than {B} when using `cu_seqlens`. "
                "Please flatten variable-length inputs before processing.")
        if cu_seqlens.ndim != 1 or cu_seqlens.shape[0] != N + 1:
            raise ValueError(f"cu_seqlens must have {N + 1} entries, one more than the rows of page_table, "
                             f"got shape {tuple(cu_seqlens.shape)}")
        if cu_seqlens.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"cu_seqlens must be int32 or int64, got {cu_seqlens.dtype}")
        if not cu_seqlens.is_contiguous():
            raise ValueError("cu_seqlens must be contiguous")
        if cu_seqlens.device != t.device:
            raise ValueError(f"cu_seqlens device {cu_seqlens.device} must match {name} ({t.device})")
    _check_strided(name, t)


_PAGE_SIZES = (16, 32, 64, 128, 256, 512, 1024)


def _plain_table(table, lens, dev) -> bool:
    """Whether these are an ordinary table and lengths on device ``dev`` that
    :func:`_check_table` accepts."""
    n = table.shape
    return (
        len(n) == 2 and n[1] > 0 and lens.shape == n[:1] and table.dtype is torch.int32 and lens.dtype is torch.int32
        and table.is_contiguous() and lens.is_contiguous() and table.get_device() == dev and lens.get_device() == dev
        and n[0] > 0
    )


def _plain_fields(k, v, table, lens, x, heads, cu) -> tuple | None:
    """The argument fields of an ordinary call on a GPU, whose cache, table,
    new tokens ``x`` (``heads`` of them, 0: any) and offsets ``cu`` the full
    checks accept, each tensor looked at once: a small call's time is the
    host's, and the checks in the order of their messages are half of it.  None
    says nothing: the full checks then accept or raise."""
    shape, s, t, dt, dev = k.shape, k.stride(), v.stride(), k.dtype, k.get_device()
    n, u, rows = x.shape, x.stride(), table.shape
    if dev < 0 or len(shape) != 4 or len(n) != 4 or v.shape != shape:
        return None
    P, size, HKV, D = shape
    s0, s1, s2, s3 = s
    t0, t1, t2, t3 = t
    u0, u1, u2, u3 = u
    kp, vp = k.data_ptr(), v.data_ptr()
    if not (
        dt in _CACHE_DTYPES and v.dtype is dt and x.dtype is dt and (D == 128 or D == 64) and size in _PAGE_SIZES
        and s3 == 1 and t3 == 1 and u3 == 1 and s0 > 0 and t0 > 0 and s1 >= D and s2 >= D and t1 >= D and t2 >= D
        and (s0 | s1 | s2 | t0 | t1 | t2 | u0 | u1 | u2) % 8 == 0 and (kp | vp | x.data_ptr()) % 16 == 0
        and P > 0 and HKV > 0 and n[0] == (rows[0] if cu is None else 1) and n[3] == D and n[1] > 0
        and (n[2] == heads if heads else n[2] > 0) and v.get_device() == dev and x.get_device() == dev
        and _plain_table(table, lens, dev)
    ):
        return None
    cu_dtype = cu_ptr = 0
    if cu is not None:
        cu_dtype = _CU_DTYPES.get(cu.dtype)
        if cu_dtype is None or cu.shape != (rows[0] + 1,) or not cu.is_contiguous() or cu.get_device() != dev:
            return None
        cu_ptr = cu.data_ptr()
    return (rows[0], n[1], n[2], HKV, D, _CACHE_DTYPES[dt], P, size, rows[1], cu_dtype, cu_ptr, table.data_ptr(), rows[1],
            lens.data_ptr(), kp, vp, s0, s1, s2, t0, t1, t2, u0, u1, u2)


def _strides(t: torch.Tensor) -> tuple[int, int, int]:
    """The first three strides; of a dimension of one element, 0."""
    s, n = t.stride(), t.shape
    return (s[0] if n[0] > 1 else 0, s[1] if n[1] > 1 else 0, s[2] if n[2] > 1 else 0)


def _fields(k, v, table, lens, x, cu_seqlens) -> tuple:
    """:func:`_plain_fields` of any call that the full checks accept."""
    P, size, HKV, D = k.shape
    N, M = table.shape
    cu_dtype = cu = 0
    if cu_seqlens is not None:
        cu_dtype = _CU_DTYPES[cu_seqlens.dtype]
        cu = cu_seqlens.data_ptr()
    return (N, x.shape[1], x.shape[2], HKV, D, _CACHE_DTYPES[k.dtype], P, size, M, cu_dtype, cu, table.data_ptr(),
            table.stride(0) if N > 1 else M, lens.data_ptr(), k.data_ptr(), v.data_ptr(), *_strides(k), *_strides(v),
            *_strides(x))


def _forward_only(name: str, *tensors: torch.Tensor) -> None:
    """The launches are outside of autograd: a gradient would be lost."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                raise NotImplementedError(f"{name} is forward only: inputs require grad")


def _launch(name: str, args: bytes, device: torch.device) -> None:
    """The entry point on the tensors' device and its current stream."""
    if torch._C._cuda_getDevice() == device.index:
        _hip.call_packed(name, args, _raw_stream(device))
        return
    with torch.cuda.device(device):
        _hip.call_packed(name, args, _raw_stream(device))


def _launch_in(name: str, args: bytes, nbytes: int, device: torch.device) -> None:
    """:func:`_launch` with a workspace of ``nbytes``, the caller's stream's
    again once the launches are queued."""
    if nbytes == 0:
        _launch(name, args + _hip.NO_WORKSPACE, device)
        return
    ws = workspace.scratch(device, nbytes)
    _launch(name, args + _hip.WORKSPACE_PACK.pack(ws.data_ptr(), nbytes), device)


def paged_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    seq_lens: torch.Tensor,
    *,
    scale: float | None = None,
    causal: bool = True,
    window: int | None = None,
    cu_seqlens: torch.Tensor | None = None,
    return_lse: bool = False,
):
    """Softmax attention of new tokens over their sequences' cached keys and
    values (the new tokens' own among them, :func:`paged_append`).

    ``q`` is ``[N, T, HQ, D]``, T new tokens of each sequence (one: a decode
    step), or with ``cu_seqlens`` ``[1, total, HQ, D]``, chunks of any lengths
    packed.  HQ is a multiple of HKV; query head h reads the cache's head
    ``h // (HQ // HKV)``; D is 64 or 128; bfloat16 or float16, like the cache.
    ``q`` may be a view (a slice of a fused projection).

    A query at position p sees the keys up to p (``causal``; else all), with
    ``window`` those above ``p - window`` only.  ``scale`` (above 0) is
    ``D ** -0.5`` by default.  Sums and the softmax are held in fp32; the
    exponentials are rounded to q's type for the product with the values.

    Returns ``o`` in q's shape and type, with ``return_lse`` also the log of
    the sum of the exponentials, fp32 ``[N, T, HQ]``.  A query that sees no
    key (an empty sequence) has o = 0 and -inf, one with a score of NaN or +inf
    NaN in both.  What the pages hold beyond ``seq_lens`` does not matter; keys and
    values before it have to be finite.
    """
    f = _plain_fields(k_cache, v_cache, page_table, seq_lens, q, 0, cu_seqlens)
    if f is None:
        _check_cache(k_cache, v_cache, page_table, seq_lens)
        _check_new("q", q, None, k_cache, page_table, cu_seqlens)
    B, T, HQ, D = q.shape
    HKV = k_cache.shape[2]
    if HQ % HKV != 0:
        raise ValueError(f"HQ must be a multiple of HKV, got HQ={HQ}, HKV={HKV}")
    if scale is None:
        scale = D ** -0.5
    if not scale > 0:
        raise ValueError(f"scale must be positive, got {scale}")
    if window is not None:
        if window < 1:
            raise ValueError(f"window must be at least 1, got {window}")
        if not causal:
            raise ValueError("window needs causal=True")
    _forward_only("paged_attention", q, k_cache, v_cache)
    if f is None:
        _require_gpu(q)
        f = _fields(k_cache, v_cache, page_table, seq_lens, q, cu_seqlens)
    device = q.device
    o = torch.empty_like(q) if q.is_contiguous() else torch.empty((B, T, HQ, D), dtype=q.dtype, device=device)
    lse = torch.empty((B, T, HQ), dtype=torch.float32, device=device) if return_lse else None
    (N, T, HQ, HKV, D, dt, P, size, M, cu_dtype, cu, table, table_stride, lens, kp, vp, s0, s1, s2, t0, t1, t2, u0, u1,
     u2) = f
    args = _hip.PAGED_PACK.pack(
        _hip.PAGED_ABI_VERSION, N, T, HQ, HKV, D, dt, P, size, M, _hip.PAGED_CAUSAL if causal else 0,
        min(window or 0, 1 << 30), scale,
        cu_dtype, cu, table, table_stride, lens, kp, vp, s0, s1, s2, t0, t1, t2, q.data_ptr(), u0, u1, u2, o.data_ptr(),
        0 if lse is None else lse.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0)
    nbytes = _hip.lib().kda_paged_attn_workspace_bytes(args + _hip.NO_WORKSPACE)
    _launch_in("kda_paged_attn_hip", args, nbytes, device)
    return (o, lse) if return_lse else o


def paged_append(
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    seq_lens: torch.Tensor,
    *,
    cu_seqlens: torch.Tensor | None = None,
) -> None:
    """Writes the new tokens' keys and values into their places in the pages.

    ``k`` and ``v`` are ``[N, T, HKV, D]`` or, with ``cu_seqlens``, packed
    ``[1, total, HKV, D]``, of the cache's type; they may be views.
    ``seq_lens`` counts the new tokens already (:func:`paged_reserve`).
    Tokens at negative positions, or whose page the table does not have, are
    left out.
    """
    f = None
    if v.shape == k.shape and v.stride() == k.stride() and v.dtype is k.dtype and (
            v.data_ptr() % 16 == 0 and v.get_device() == k.get_device()):
        f = _plain_fields(k_cache, v_cache, page_table, seq_lens, k, k_cache.shape[2], cu_seqlens)
    if f is None:
        _check_cache(k_cache, v_cache, page_table, seq_lens)
        for name, t in (("k", k), ("v", v)):
            _check_new(name, t, k_cache.shape[2], k_cache, page_table, cu_seqlens)
        if v.shape != k.shape:
            raise ValueError(f"v.shape {tuple(v.shape)} must match k {tuple(k.shape)}")
    _forward_only("paged_append", k, v, k_cache, v_cache)
    if f is None:
        _require_gpu(k)
        f = _fields(k_cache, v_cache, page_table, seq_lens, k, cu_seqlens) + _strides(v)
    (N, T, HQ, HKV, D, dt, P, size, M, cu_dtype, cu, table, table_stride, lens, kp, vp, s0, s1, s2, t0, t1, t2, u0, u1,
     u2), w = f[:25], f[25:] or f[22:]
    _launch("kda_paged_append_hip", _hip.PAGED_PACK.pack(
        _hip.PAGED_ABI_VERSION, N, T, HQ, HKV, D, dt, P, size, M, 0, 0, 1.0, cu_dtype, cu, table, table_stride, lens, kp,
        vp, s0, s1, s2, t0, t1, t2, 0, 0, 0, 0, 0, 0, k.data_ptr(), v.data_ptr(), u0, u1, u2, *w) + _hip.NO_WORKSPACE,
        k.device)


def _pools(pools) -> list[torch.Tensor]:
    """The pools of a call, checked: ``[..., P, a, b, c]`` each."""
    ts = [pools] if isinstance(pools, torch.Tensor) else list(pools)
    if not 1 <= len(ts) <= _hip.PAGED_MAX_POOLS:
        raise ValueError(f"between 1 and {_hip.PAGED_MAX_POOLS} pools, got {len(ts)}")
    P = ts[0].shape[-4] if ts[0].ndim >= 4 else 0
    for i, t in enumerate(ts):
        if t.ndim < 4:
            raise ValueError(f"pool {i} must be at least 4D [..., P, a, b, c], got shape {tuple(t.shape)}")
        if not t.is_contiguous():
            raise ValueError(f"pool {i} must be contiguous")
        if t.numel() == 0:
            raise ValueError(f"pool {i} dimensions must be positive, got shape {tuple(t.shape)}")
        if t.shape[-4] != P:
            raise ValueError(f"pool {i} must have {P} pages like the first, got {t.shape[-4]}")
        if i > 0 and t.device != ts[0].device:
            raise ValueError(f"pool {i} device {t.device} must match the first's ({ts[0].device})")
        if t.data_ptr() % 16 or t.stride(-4) * t.element_size() % 16:
            raise ValueError(f"pool {i} must be 16-byte aligned, its pages multiples of 16 bytes")
    return ts


_NO_POOLS = (0,) * (3 * _hip.PAGED_MAX_POOLS)


def _pool_fields(pools, P) -> tuple:
    out = ()
    for t in pools:
        size = t.element_size()
        page = t.stride(-4) * size
        out += (t.data_ptr(), t.numel() * size // (P * page), page)
    return out + _NO_POOLS[len(out):]


def _pack(P, page_size, F, num_pools, pools, table, table_stride=0, N=0, M=0, lens=0, refs=0, src=0, dst=0, more=0, ok=0,
          out_table=0, out_refs=0, out_live=0) -> bytes:
    """The packed arguments of a call on the pages, up to the workspace
    (pointers, 0 for none)."""
    return _hip.PAGES_PACK.pack(
        _hip.PAGED_ABI_VERSION, N, M, P, page_size, F, num_pools, 0, *pools, table, table_stride, lens, refs, src, dst,
        more, ok, out_table, out_refs, out_live)


def _check_refs(page_refs, device) -> None:
    _int32("page_refs", page_refs, 1, device)
    if page_refs.shape[0] < 1:
        raise ValueError("page_refs must not be empty")
    if page_refs.data_ptr() % 16:
        raise ValueError("page_refs must be 16-byte aligned")


def _check_rows(pairs, device) -> None:
    for name, t in pairs:
        _int32(name, t, 1, device)
        if t.shape[0] != pairs[0][1].shape[0]:
            raise ValueError(f"{name} must have {pairs[0][1].shape[0]} entries like {pairs[0][0]}, got {t.shape[0]}")


def _plain_rows(a, b, dev) -> bool:
    """Whether these are ordinary int32 rows on GPU ``dev`` that
    :func:`_check_rows` accepts (as for :func:`_plain_fields`)."""
    n = a.shape
    return (len(n) == 1 and b.shape == n and a.dtype is torch.int32 and b.dtype is torch.int32 and a.get_device() == dev
            and b.get_device() == dev and a.is_contiguous() and b.is_contiguous())


def _check_counts(page_table, seq_lens, page_refs) -> int:
    """Table, lengths and counts of one cache; their GPU, -1 for none."""
    dev = page_table.get_device()
    if not (dev >= 0 and _plain_table(page_table, seq_lens, dev) and page_refs.dtype is torch.int32
            and page_refs.ndim == 1 and page_refs.get_device() == dev and page_refs.is_contiguous()
            and page_refs.data_ptr() % 16 == 0 and page_refs.shape[0] > 0):
        _check_table(page_table, seq_lens, page_table.device)
        _check_refs(page_refs, page_table.device)
    return dev


def paged_reserve(
    page_table: torch.Tensor,
    seq_lens: torch.Tensor,
    page_refs: torch.Tensor,
    new_tokens: torch.Tensor,
    page_size: int,
) -> torch.Tensor:
    """Room for ``new_tokens[n]`` (int32 ``[N]``) more tokens of every
    sequence: first the pages that its row holds past its length, then the
    lowest free ones, in the sequences' order, until they run out;
    ``seq_lens`` grows by as many.

    Returns a bool ``[N]``: False for a sequence whose pages cannot all be
    had, or do not fit its row; it keeps what it has.  Once pages could not all
    be had, later sequences get none.
    """
    dev = _check_counts(page_table, seq_lens, page_refs)
    if not _plain_rows(seq_lens, new_tokens, dev):
        _check_rows([("seq_lens", seq_lens), ("new_tokens", new_tokens)], page_table.device)
    _check_page_size(page_size)
    _require_gpu(page_table)
    ok = seq_lens.new_empty(seq_lens.shape[0], dtype=torch.bool)
    N, M = page_table.shape
    _launch("kda_pages_reserve_hip", _pack(
        page_refs.shape[0], page_size, 0, 0, _NO_POOLS, page_table.data_ptr(), page_table.stride(0) if N > 1 else M, N, M,
        seq_lens.data_ptr(), page_refs.data_ptr(), 0, 0, new_tokens.data_ptr(), ok.data_ptr()) + _hip.NO_WORKSPACE,
        page_table.device)
    return ok


def paged_free(
    page_table: torch.Tensor,
    seq_lens: torch.Tensor,
    page_refs: torch.Tensor,
    rows: torch.Tensor,
) -> None:
    """The sequences ``rows`` (int32) end: their pages lose a holder each,
    their entries become -1, their lengths 0."""
    dev = _check_counts(page_table, seq_lens, page_refs)
    if not _plain_rows(rows, rows, dev):
        _check_rows([("rows", rows)], page_table.device)
    _require_gpu(page_table)
    N, M = page_table.shape
    _launch("kda_pages_free_hip", _pack(
        page_refs.shape[0], 16, rows.shape[0], 0, _NO_POOLS, page_table.data_ptr(),
        page_table.stride(0) if N > 1 else M, N, M, seq_lens.data_ptr(), page_refs.data_ptr(), 0, rows.data_ptr())
        + _hip.NO_WORKSPACE, page_table.device)


def paged_fork(
    pools,
    page_table: torch.Tensor,
    seq_lens: torch.Tensor,
    page_refs: torch.Tensor,
    src: torch.Tensor,
    dst: torch.Tensor,
    *,
    page_size: int | None = None,
) -> torch.Tensor:
    """Row ``dst[i]`` (new or freed) becomes a copy of row ``src[i]`` (int32): whole
    pages are shared, the tokens of a last partial page copied, in every pool,
    to the lowest free page not taken by an earlier fork.

    ``pools`` is a tensor ``[..., P, page_size, HKV, D]`` or a sequence of
    them (up to 8): keys and values of all layers in one, or apart.  With
    another order of a page's dimensions (``[..., P, HKV, page_size, D]``)
    give ``page_size``.  Rows of ``dst`` are distinct and none is in ``src``;
    a row of ``src`` may be forked several times.

    Returns a bool per fork: False where no page was left; the row stays empty.
    """
    ts = _pools(pools)
    device = ts[0].device
    dev = _check_counts(page_table, seq_lens, page_refs)
    if dev != ts[0].get_device():
        raise ValueError(f"page_table device {page_table.device} must match ({device})")
    if not _plain_rows(src, dst, dev):
        _check_rows([("src", src), ("dst", dst)], device)
    page_size = ts[0].shape[-3] if page_size is None else page_size
    _check_page_size(page_size)
    P, F = ts[0].shape[-4], src.shape[0]
    if page_refs.shape[0] != P:
        raise ValueError(f"page_refs must have one entry a page, {P}, got {page_refs.shape[0]}")
    _forward_only("paged_fork", *ts)
    _require_gpu(ts[0])
    ok = src.new_empty(F, dtype=torch.bool)
    N, M = page_table.shape
    _launch("kda_pages_fork_hip", _pack(
        P, page_size, F, len(ts), _pool_fields(ts, P), page_table.data_ptr(), page_table.stride(0) if N > 1 else M, N, M,
        seq_lens.data_ptr(), page_refs.data_ptr(), src.data_ptr(), dst.data_ptr(), 0, ok.data_ptr()) + _hip.NO_WORKSPACE,
        device)
    return ok


def paged_copy(pools, src: torch.Tensor, dst: torch.Tensor) -> None:
    """``pool[..., dst[i], :, :, :] = pool[..., src[i], :, :, :]`` for every
    pool, ``[..., P, a, b, c]``, in one launch.

    Pages of a cache, or whatever else goes along with a sequence: recurrent
    states ``[layers, rows, HV, 128, 128]`` are a pool of ``rows`` pages.
    Pairs outside ``[0, P)`` are left out; no page is in ``src`` and in
    ``dst``, or in ``dst`` twice.
    """
    ts = _pools(pools)
    device = ts[0].device
    if not _plain_rows(src, dst, ts[0].get_device()):
        _check_rows([("src", src), ("dst", dst)], device)
    _forward_only("paged_copy", *ts)
    _require_gpu(ts[0])
    P = ts[0].shape[-4]
    _launch("kda_pages_copy_hip", _pack(P, 16, src.shape[0], len(ts), _pool_fields(ts, P), 0, src=src.data_ptr(),
                                        dst=dst.data_ptr()) + _hip.NO_WORKSPACE, device)


def paged_compact(
    pools,
    page_table: torch.Tensor,
    page_refs: torch.Tensor,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Moves the held pages into the first ``live`` places of every pool,
    live being their number: the i-th held page at or above ``live`` goes to
    the i-th free place below it.

    Returns ``(page_table, page_refs, live)``, new tensors (live: int32
    ``[1]``).  The old table and counts stay as they are, and the pages moved
    away from keep their contents: a launch on another stream that still reads
    by the old table stays right until those pages are handed out again.
    """
    ts = _pools(pools)
    device = ts[0].device
    P = ts[0].shape[-4]
    _int32("page_table", page_table, 2, device)
    if page_table.shape[0] < 1 or page_table.shape[1] < 1:
        raise ValueError(f"page_table dimensions must be positive, got shape {tuple(page_table.shape)}")
    if page_table.shape[0] > 1 and page_table.stride(0) < page_table.shape[1]:
        raise ValueError("rows of page_table must not overlap")
    _check_refs(page_refs, device)
    if page_refs.shape[0] != P:
        raise ValueError(f"page_refs must have one entry a page, {P}, got {page_refs.shape[0]}")
    _forward_only("paged_compact", *ts)
    _require_gpu(ts[0])
    N, M = page_table.shape
    table = torch.empty_like(page_table) if page_table.is_contiguous() else page_table.new_empty((N, M))
    refs = torch.empty_like(page_refs)
    live = page_refs.new_empty(1)
    args = _pack(P, 16, 0, len(ts), _pool_fields(ts, P), page_table.data_ptr(), page_table.stride(0) if N > 1 else M, N, M,
                 0, page_refs.data_ptr(), out_table=table.data_ptr(), out_refs=refs.data_ptr(), out_live=live.data_ptr())
    _launch_in("kda_pages_compact_hip", args, _hip.lib().kda_pages_workspace_bytes(args + _hip.NO_WORKSPACE), device)
    return table, refs, live
