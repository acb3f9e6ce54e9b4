"""Attention of groups that share their first tokens: checks of arguments and
the C ABI (CPU only)."""

from __future__ import annotations

import ctypes
import re
import shutil
import subprocess

import pytest
import torch

from kda_bt16 import _hip, paged_attention_shared
from test_paged_capi import FAKE, HEADER, _text, fake_pointers, paged

BF16 = torch.bfloat16


def _i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def call(**change):
    a = dict(q=torch.zeros(2, 3, 4, 64, dtype=BF16), k_cache=torch.zeros(5, 16, 2, 64, dtype=BF16),
             v_cache=torch.zeros(5, 16, 2, 64, dtype=BF16), page_table=_i32(2, 4), seq_lens=_i32(2), cu_groups=_i32(3),
             shared_lens=_i32(2))
    kw = {k: change.pop(k) for k in list(change) if k not in a}
    a.update(change)
    return paged_attention_shared(*a.values(), **kw)


def test_wants_a_gpu():
    with pytest.raises(ValueError, match="runs on a ROCm GPU"):
        call()


@pytest.mark.parametrize("change,error,match", [
    (dict(cu_groups=torch.zeros(3, dtype=torch.int64)), TypeError, "cu_groups must be int32"),
    (dict(cu_groups=_i32(3, 1)), ValueError, "cu_groups must be 1D"),
    (dict(cu_groups=_i32(6)[::2]), ValueError, "cu_groups must be contiguous"),
    (dict(shared_lens=torch.zeros(2)), TypeError, "shared_lens must be int32"),
    (dict(cu_groups=_i32(2)), ValueError, "one entry more than shared_lens"),
    (dict(cu_groups=_i32(1), shared_lens=_i32(0)), ValueError, "of one at least"),
    (dict(q=torch.zeros(2, 3, 3, 64, dtype=BF16)), ValueError, "HQ must be a multiple"),
    (dict(q=torch.zeros(2, 3, 4, 64)), TypeError, "q must be"),
    (dict(scale=0.0), ValueError, "scale must be positive"),
    (dict(page_table=_i32(2, 4).to(torch.int64)), TypeError, "page_table must be int32"),
    (dict(cu_seqlens=_i32(3)), ValueError, "expected to be 1 rather than 2"),
    (dict(k_cache=torch.zeros(5, 16, 2, 64, dtype=BF16, requires_grad=True)), NotImplementedError,
     "paged_attention_shared is forward only"),
])
def test_refusals(change, error, match):
    with pytest.raises(error, match=match):
        call(**change)


def test_struct_matches_the_header():
    for cls in (_hip.KdaPagedSharedArgs, _hip.KdaPagedSinksArgs):
        name = cls.__name__
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), _text(), re.S).group(1)
        names = []
        for decl in filter(None, (d.strip() for d in body.split(";"))):
            names += [n.strip().lstrip("*") for n in re.sub(r"^.*?\b(?=\w+\s*(,|$))", "", decl).split(",")]
        assert names == [f for f, _ in cls._fields_]


@pytest.mark.skipif(shutil.which("gcc") is None, reason="no C compiler")
def test_c_compiler_sees_the_same_layout(tmp_path):
    want, lines = [], []
    for cls in (_hip.KdaPagedSharedArgs, _hip.KdaPagedSinksArgs):
        lines.append(f'printf("%zu\\n", sizeof({cls.__name__}));')
        lines += [f'printf("%zu\\n", offsetof({cls.__name__}, {f}));' for f, _ in cls._fields_]
        want += [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "kda_paged_hip.h"\nint main(void) {\n'
                   + "\n".join(lines) + "\nreturn 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", f"-I{HEADER.parent}", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()
    assert [int(x) for x in out] == want


def shared(base=None, **change):
    tail = dict(cu_groups=FAKE, shared_lens=FAKE, num_groups=2, reserved=0) | change
    return _hip.KdaPagedSharedArgs(paged(**dict(flags=_hip.PAGED_CAUSAL) | (base or {})), *tail.values())


def test_packed_arguments_are_the_struct():
    a = shared()
    assert bytes(a) == bytes(a.paged) + _hip.SHARED_PACK.pack(FAKE, FAKE, 2, 0)


def test_workspace_sizes():
    f, plain = _hip.lib().kda_paged_attn_shared_workspace_bytes, _hip.lib().kda_paged_attn_workspace_bytes
    assert f(None) == 0
    # one sequence, whole row tiles, more sequences than a plan holds, rows of few keys
    # (112 MB of keys and values together, 224 with more than 16 rows a sequence):
    # as without groups
    wide = dict(M=8000, table_stride=8000)
    for base in (dict(N=1, **wide), dict(T=128, **wide), dict(N=2049, **wide), dict(), dict(M=3583, table_stride=3583),
                 dict(T=16, M=6000, table_stride=6000)):
        a = shared(base)
        assert f(ctypes.byref(a)) == plain(ctypes.byref(a.paged)), base
    for base in (dict(N=2048), dict(T=127, **wide), dict(M=3584, table_stride=3584), dict(T=16, **wide)):
        a = shared(base)
        assert f(ctypes.byref(a)) != plain(ctypes.byref(a.paged)), base
    # 8 sequences of a token, 8 / 2 heads: rows of both kinds (2 * 32 * 2, and 3 for each of 10 records and
    # head), 1024 places of 32 rows, in rows of D + 2 floats; the plan of 10 records and 8 tokens
    rows = 2 * 8 * 4 * 2 + 3 * 10 * 2 + 2 * 512 * 32
    got = f(ctypes.byref(shared(dict(N=8, HQ=8, q_row=1024, q_token=1024, **wide))))
    assert got == (rows + 3) // 4 * 4 * 130 * 4 + (16 + 10 * 16 + 8) * 4


def test_workspace_of_dense_rows_past_a_row_tile():
    """More than 128 rows a sequence: one by one, in what paged_attention takes."""
    f, plain = _hip.lib().kda_paged_attn_shared_workspace_bytes, _hip.lib().kda_paged_attn_workspace_bytes
    for heads, T in ((4, 65), (4, 100), (4, 127), (16, 17), (16, 31), (260, 1)):
        base = dict(T=T, HQ=heads, q_row=T * heads * 128, q_token=heads * 128, M=8000, table_stride=8000)
        a = shared(base)
        assert 0 <= f(ctypes.byref(a)) - plain(ctypes.byref(a.paged)) <= 1 << 16, base
    # (65 to 128 row tiles of 256: in the plan's finer parts)
    for N, more in ((32, False), (33, True), (64, True), (65, False)):
        a = shared(base | dict(N=N))
        assert (f(ctypes.byref(a)) - plain(ctypes.byref(a.paged)) > 1 << 16) == more, N


def test_workspace_of_tables_that_one_launch_takes_whole():
    """Rows of up to 768 keys, decode and drafts, up to two rounds of row tiles: as
    without groups, which takes no workspace; else a plan's."""
    f = _hip.lib().kda_paged_attn_shared_workspace_bytes
    small = dict(N=512, M=48, table_stride=48)
    for base in (small, small | dict(T=16), small | dict(N=400)):
        assert f(ctypes.byref(shared(base))) == 0, base
    for base in (small | dict(M=49, table_stride=49), small | dict(N=513), small | dict(T=17),
                 small | dict(cu_seqlens=FAKE, T=512, cu_seqlens_dtype=_hip.DTYPE_I32)):
        assert f(ctypes.byref(shared(base))) > 0, base


@fake_pointers
def test_argument_checks():
    f = _hip.lib().kda_paged_attn_shared_hip
    assert f(None, None) == -1
    for bad in (dict(num_groups=0), dict(num_groups=-1), dict(cu_groups=0), dict(shared_lens=0), dict(cu_groups=FAKE + 2),
                dict(shared_lens=FAKE + 1)):
        assert f(ctypes.byref(shared(**bad)), None) == -1, bad
    assert f(ctypes.byref(shared(dict(flags=0))), None) == -2
    assert f(ctypes.byref(shared(dict(window=5))), None) == -2
    assert f(ctypes.byref(shared(dict(D=96))), None) == -2 and f(ctypes.byref(shared(dict(abi_version=4))), None) == -5
    assert f(ctypes.byref(shared()), None) == -3  # no workspace
    assert f(ctypes.byref(shared(dict(workspace=FAKE, workspace_bytes=1 << 12))), None) == -3
