"""The paged cache's C ABI (CPU only): include/kda_paged_hip.h against the
binding and a C compiler, and the argument checks that come before any
launch."""

from __future__ import annotations

import ctypes
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from kda_bt16 import _hip

ROOT = Path(__file__).resolve().parents[1]
HEADER = ROOT / "include" / "kda_paged_hip.h"
STRUCTS = {"KdaPagedArgs": _hip.KdaPagedArgs, "KdaPagePool": _hip.KdaPagePool, "KdaPagesArgs": _hip.KdaPagesArgs}

# Stand-in pointers reach launching entry points only where no GPU is present:
# a check that regressed could launch a kernel on them.
fake_pointers = pytest.mark.skipif(torch.cuda.is_available(), reason="stand-in device pointers need a box without a GPU")
FAKE = 1 << 40


def _text():
    return re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)


def test_header_declares_the_binding_symbols():
    assert sorted(set(re.findall(r"\b(kda_\w+)\s*\(", _text()))) == sorted(_hip.PAGED_SYMBOLS)
    for name in _hip.PAGED_SYMBOLS:
        assert hasattr(_hip.lib(), name)


@pytest.mark.parametrize("name", STRUCTS)
def test_struct_fields_match_the_header(name):
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), _text(), re.S).group(1)
    names = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        decl = re.sub(r"\[\w+\]", "", decl)
        names += [n.strip().lstrip("*") for n in re.sub(r"^.*?\b(?=\w+\s*(,|$))", "", decl).split(",")]
    assert names == [f for f, _ in STRUCTS[name]._fields_]


@pytest.mark.skipif(shutil.which("gcc") is None, reason="no C compiler")
def test_c_compiler_sees_the_same_layout(tmp_path):
    lines = []
    for name, cls in STRUCTS.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "kda_paged_hip.h"\nint main(void) {\n'
                   + "\n".join(lines) + "\nreturn 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Wextra", "-Werror", "-pedantic", f"-I{HEADER.parent}", str(src), "-o",
                    str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    got = dict(line.split() for line in out.splitlines())
    for name, cls in STRUCTS.items():
        assert int(got[name]) == ctypes.sizeof(cls)
        for f, _ in cls._fields_:
            assert int(got[f"{name}.{f}"]) == getattr(cls, f).offset, f


def test_packed_arguments_are_the_structs():
    for cls, pack in ((_hip.KdaPagedArgs, _hip.PAGED_PACK), (_hip.KdaPagesArgs, _hip.PAGES_PACK)):
        values, flat = [], []
        for i, (_, t) in enumerate(cls._fields_[:-2]):
            if issubclass(t, ctypes.Array):
                items = [(1000 + 3 * j, 1001 + 3 * j, 1002 + 3 * j) for j in range(t._length_)]
                values.append(t(*items))
                flat += [x for item in items for x in item]
            else:
                values.append(i + 1)
                flat.append(i + 1)
        packed = pack.pack(*flat) + _hip.WORKSPACE_PACK.pack(77, 88)
        assert packed == bytes(cls(*values, 77, 88))


def test_constants_match_the_binding():
    consts = dict(re.findall(r"#define\s+(KDA_PAGED_\w+)\s+\(?([^\s/)]+)", HEADER.read_text()))
    assert int(consts["KDA_PAGED_ABI_VERSION"]) == _hip.PAGED_ABI_VERSION == _hip.lib().kda_paged_abi_version()
    assert int(consts["KDA_PAGED_BF16"]) == _hip.PAGED_BF16 and int(consts["KDA_PAGED_FP16"]) == _hip.PAGED_FP16
    assert int(consts["KDA_PAGED_MAX_POOLS"]) == _hip.PAGED_MAX_POOLS
    assert consts["KDA_PAGED_CAUSAL"] == "1u" and _hip.PAGED_CAUSAL == 1


def paged(**change):
    a = _hip.KdaPagedArgs()
    base = dict(abi_version=_hip.PAGED_ABI_VERSION, N=2, T=1, HQ=4, HKV=2, D=128, P=10, page_size=16, M=100, scale=0.1,
                page_table=FAKE, table_stride=100, seq_lens=FAKE, k=FAKE, v=FAKE, k_page=4096, k_token=256, k_head=128,
                v_page=4096, v_token=256, v_head=128, q=FAKE, q_row=512, q_token=512, q_head=128, o=FAKE, new_k=FAKE,
                new_v=FAKE, nk_row=256, nk_token=256, nk_head=128, nv_row=256, nv_token=256, nv_head=128)
    for name, value in (base | change).items():
        setattr(a, name, value)
    return a


def pages(**change):
    a = _hip.KdaPagesArgs()
    base = dict(abi_version=_hip.PAGED_ABI_VERSION, N=2, M=10, P=20, page_size=16, F=1, num_pools=1, page_table=FAKE,
                table_stride=10, seq_lens=FAKE, page_refs=FAKE, src=FAKE, dst=FAKE, new_tokens=FAKE, ok=FAKE,
                out_table=FAKE, out_refs=FAKE, out_live=FAKE, workspace=FAKE, workspace_bytes=1 << 20)
    a.pools[0] = (FAKE, 3, 4096)
    for name, value in (base | change).items():
        if name == "pool":
            a.pools[0] = value
        else:
            setattr(a, name, value)
    return a


def test_workspace_sizes():
    f = _hip.lib().kda_paged_attn_workspace_bytes
    assert f(None) == 0 and f(ctypes.byref(paged(D=96))) == 0
    assert f(ctypes.byref(paged(M=48, table_stride=48))) == 0  # 768 keys: one launch, no parts
    few = f(ctypes.byref(paged()))
    assert few == 2 * 512 * 32 * 130 * 4
    assert f(ctypes.byref(paged(D=64))) == 2 * 512 * 32 * 66 * 4
    # a chunk whose row tiles do not fill the card: parts of 256 rows too
    assert f(ctypes.byref(paged(T=400))) == few + 256 * 256 * 130 * 4
    assert f(ctypes.byref(paged(T=400, N=100))) == 0  # enough row tiles, taken whole
    g = _hip.lib().kda_pages_workspace_bytes
    assert g(None) == 0 and g(ctypes.byref(pages(P=0))) == 0
    assert g(ctypes.byref(pages(P=5000))) == (4 * (3 * 5000 + 1 + 2) + 255) // 256 * 256


@fake_pointers
@pytest.mark.parametrize("name", ["kda_paged_attn_hip", "kda_paged_append_hip"])
def test_paged_argument_checks(name):
    f = getattr(_hip.lib(), name)
    assert f(None, None) == -1
    assert f(ctypes.byref(paged(abi_version=99)), None) == -5
    for bad in (dict(N=0), dict(T=0), dict(HKV=0), dict(P=0), dict(M=0), dict(dtype=2), dict(page_table=0),
                dict(seq_lens=0), dict(k=0), dict(v=0), dict(k=FAKE + 8), dict(v=FAKE + 2), dict(page_table=FAKE + 2),
                dict(table_stride=99), dict(k_head=4), dict(v_page=-8), dict(cu_seqlens=FAKE, cu_seqlens_dtype=0),
                dict(cu_seqlens=FAKE + 4, cu_seqlens_dtype=_hip.DTYPE_I64)):
        assert f(ctypes.byref(paged(**bad)), None) == -1, bad
    for bad in (dict(D=96), dict(page_size=24), dict(page_size=8), dict(page_size=2048), dict(k_token=120),
                dict(v_token=1 << 31), dict(k_page=1 << 31), dict(M=1 << 27, table_stride=1 << 27)):
        assert f(ctypes.byref(paged(**bad)), None) == -2, bad
    with pytest.raises(_hip.KdaHipError, match="code -2"):
        _hip.call_packed(name, bytes(paged(D=96)), 0)


@fake_pointers
def test_attention_and_append_checks_of_their_own():
    f = _hip.lib().kda_paged_attn_hip
    for bad in (dict(HQ=0), dict(HQ=3), dict(window=-1), dict(scale=0.0), dict(scale=float("nan")), dict(q=0), dict(o=0),
                dict(q=FAKE + 8), dict(q_head=4), dict(lse=FAKE + 2)):
        assert f(ctypes.byref(paged(**bad)), None) == -1, bad
    assert f(ctypes.byref(paged(window=4)), None) == -2  # without causal
    assert f(ctypes.byref(paged(N=1 << 20, M=1 << 14, table_stride=1 << 14)), None) == -2  # tiles past 32 bits
    assert f(ctypes.byref(paged(N=1 << 20, T=1 << 10)), None) == -2  # rows past 32 bits
    assert f(ctypes.byref(paged()), None) == -3  # no workspace
    assert f(ctypes.byref(paged(workspace=FAKE + 16, workspace_bytes=1 << 30)), None) == -3
    assert f(ctypes.byref(paged(workspace=FAKE, workspace_bytes=1 << 10)), None) == -3
    g = _hip.lib().kda_paged_append_hip
    for bad in (dict(new_k=0), dict(new_v=0), dict(new_v=FAKE + 8), dict(nk_head=4), dict(nv_token=-8)):
        assert g(ctypes.byref(paged(**bad)), None) == -1, bad
    assert g(ctypes.byref(paged(N=1 << 20, T=1 << 10)), None) == -2


@fake_pointers
def test_page_argument_checks():
    lib = _hip.lib()
    every = ("reserve", "free", "fork", "copy", "compact")
    calls = {n: getattr(lib, f"kda_pages_{n}_hip") for n in every}

    def rc(name, **bad):
        return calls[name](ctypes.byref(pages(**bad)), None)

    for name in every:
        assert calls[name](None, None) == -1
        assert rc(name, abi_version=7) == -5
        assert rc(name, P=0) == -1 and rc(name, F=-1) == -1
    for name in ("fork", "copy", "compact"):
        for bad in (dict(num_pools=0), dict(num_pools=9), dict(pool=(0, 3, 4096)), dict(pool=(FAKE + 8, 3, 4096)),
                    dict(pool=(FAKE, 0, 4096)), dict(pool=(FAKE, 3, 24)), dict(pool=(FAKE, 3, 0))):
            assert rc(name, **bad) == -1, (name, bad)
    for name in ("reserve", "free", "fork", "compact"):
        for bad in (dict(N=0), dict(M=0), dict(page_table=0), dict(table_stride=9), dict(page_refs=0),
                    dict(page_refs=FAKE + 4)):
            assert rc(name, **bad) == -1, (name, bad)
    for name in ("reserve", "free", "fork"):
        assert rc(name, seq_lens=0) == -1
        assert rc(name, page_size=48) == -2
        assert rc(name, M=1 << 27, table_stride=1 << 27) == -2
    assert rc("reserve", new_tokens=0) == -1 and rc("reserve", ok=0) == -1
    assert rc("free", dst=0) == -1 and rc("fork", src=0) == -1 and rc("fork", ok=0) == -1 and rc("copy", dst=0) == -1
    for bad in (dict(out_table=0), dict(out_refs=0), dict(out_live=0), dict(out_live=FAKE + 2)):
        assert rc("compact", **bad) == -1
    assert rc("compact", workspace=0) == -3 and rc("compact", workspace_bytes=64) == -3
    # nothing to do
    for name in ("free", "fork", "copy"):
        assert rc(name, F=0, src=0, dst=0) == 0
