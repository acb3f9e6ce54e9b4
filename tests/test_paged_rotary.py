"""The append with the position rotation: its checks of arguments and its C
ABI (CPU only)."""

from __future__ import annotations

import ctypes
import re
import shutil
import subprocess

import pytest
import torch

from kda_bt16 import _hip, paged_append_rotary
from kda_bt16.paged import _apart
from test_paged_capi import FAKE, HEADER, _text, fake_pointers, paged

BF16 = torch.bfloat16


def _i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def call(**change):
    a = dict(q=torch.zeros(2, 3, 4, 64, dtype=BF16), k=torch.zeros(2, 3, 2, 64, dtype=BF16),
             v=torch.zeros(2, 3, 2, 64, dtype=BF16), k_cache=torch.zeros(5, 16, 2, 64, dtype=BF16),
             v_cache=torch.zeros(5, 16, 2, 64, dtype=BF16), page_table=_i32(2, 4), seq_lens=_i32(2),
             inv_freq=torch.zeros(32))
    kw = {k: change.pop(k) for k in list(change) if k not in a}
    a.update(change)
    return paged_append_rotary(*a.values(), **kw)


def test_wants_a_gpu():
    for kw in ({}, dict(out=torch.zeros(2, 3, 4, 64, dtype=BF16))):
        with pytest.raises(ValueError, match="runs on a ROCm GPU"):
            call(**kw)


_BUF = torch.zeros(2, 3, 8, 64, dtype=BF16)


@pytest.mark.parametrize("change,error,match", [
    (dict(q=torch.zeros(3, 4, 64, dtype=BF16)), ValueError, "same tokens|q must be 4D"),
    (dict(q=torch.zeros(2, 3, 4, 64)), TypeError, "q must be torch.bfloat16 like the cache"),
    (dict(q=torch.zeros(2, 4, 4, 64, dtype=BF16)), ValueError, "same tokens"),
    (dict(k=torch.zeros(2, 3, 1, 64, dtype=BF16), v=torch.zeros(2, 3, 1, 64, dtype=BF16)), ValueError, "the cache's 2 heads"),
    (dict(v=torch.zeros(2, 3, 1, 64, dtype=BF16)), ValueError, "same heads"),
    (dict(v=torch.zeros(2, 3, 2, 64)), TypeError, "v must be"),
    (dict(k=torch.zeros(2, 3, 2, 68, dtype=BF16)[..., :64]), ValueError, "strides multiples of 8"),
    (dict(k_cache=torch.zeros(5, 24, 2, 64, dtype=BF16), v_cache=torch.zeros(5, 24, 2, 64, dtype=BF16)), ValueError,
     "power of two"),
    (dict(page_table=torch.zeros(2, 4)), TypeError, "page_table must be int32"),
    (dict(inv_freq=torch.zeros(32, dtype=torch.float64)), ValueError, "inv_freq must be contiguous 1D float32"),
    (dict(inv_freq=torch.zeros(2, 16)), ValueError, "inv_freq must be contiguous 1D"),
    (dict(inv_freq=torch.zeros(64)[::2]), ValueError, "inv_freq must be contiguous"),
    (dict(inv_freq=torch.zeros(0)), ValueError, "multiple of 16 from 16 to the head size 64, got 0"),
    (dict(inv_freq=torch.zeros(12)), ValueError, "got 24"),
    (dict(inv_freq=torch.zeros(40)), ValueError, "got 80"),
    (dict(cu_seqlens=_i32(3)), ValueError, "expected to be 1 rather than 2"),
    (dict(out=torch.zeros(2, 3, 2, 64, dtype=BF16)), ValueError, "out must have the cache's 4 heads"),
    (dict(out=torch.zeros(2, 3, 4, 64)), TypeError, "out must be"),
    (dict(out=torch.zeros(2, 1, 4, 64, dtype=BF16).expand(2, 3, 4, 64)), ValueError, "out's elements must not overlap"),
    (dict(out=torch.zeros(2000, dtype=BF16).as_strided((2, 3, 4, 64), (256, 64, 64, 1))), ValueError, "must not overlap"),
    (dict(q=_BUF[:, :, :4], out=_BUF[:, :, 4:]), ValueError, "q itself or of other storage"),
    (dict(q=_BUF[:, :, :4], out=_BUF[:, :, 2:6]), ValueError, "q itself or of other storage"),
])
def test_refusals(change, error, match):
    with pytest.raises(error, match=match):
        call(**change)


def test_in_place_on_a_broadcast_input_is_refused():
    q = torch.zeros(2, 1, 4, 64, dtype=BF16).expand(2, 3, 4, 64)
    with pytest.raises(ValueError, match="must not overlap"):
        call(q=q, out=q)


@pytest.mark.parametrize("k,v", [(slice(0, 2), slice(6, 8)), (slice(4, 6), slice(3, 5)), (slice(2, 4), slice(2, 4))])
def test_in_place_on_keys_or_values_is_refused(k, v):
    q = _BUF[:, :, :4]
    with pytest.raises(ValueError, match="k and v must lie apart"):
        call(q=q, out=q, k=_BUF[:, :, k], v=_BUF[:, :, v])


@pytest.mark.parametrize("shape,order", [((2, 3, 8, 64), (0, 1, 2, 3)), ((2, 8, 3, 64), (0, 2, 1, 3)), ((8, 2, 3, 64), (1, 2, 0, 3)),
                                         ((2, 3, 8, 64), None)])
def test_in_place_beside_keys_and_values(shape, order):
    """Slices of one projection, tokens or heads outside, and tensors of their
    own, go on to the launch."""
    buf = torch.zeros(shape, dtype=BF16)
    buf = buf if order is None else buf.permute(order)
    for parts in ((slice(0, 4), slice(4, 6), slice(6, 8)), (slice(2, 6), slice(0, 2), slice(6, 8)), (slice(4, 8), slice(0, 2), slice(2, 4))):
        q, k, v = (buf[:, :, x] if order else buf[:, :, x].contiguous() for x in parts)
        with pytest.raises(ValueError, match="runs on a ROCm GPU"):
            call(q=q, out=q, k=k, v=v)


@pytest.mark.parametrize("shape,order,at", [
    ((3, 2, 8, 64), (1, 0, 2, 3), 2), ((8, 3, 2, 64), (2, 1, 0, 3), 2), ((3, 8, 2, 64), (2, 0, 1, 3), 2),
    ((2, 3, 2, 3, 64), None, 3), ((3, 2, 2, 3, 64), (1, 0, 2, 3, 4), 3), ((2, 3, 3, 2, 64), None, 2)])
def test_in_place_beside_keys_and_values_in_any_order(shape, order, at):
    """Slices of one projection whose tokens stand outside of the rows (time
    first), or of whose heads each has its query, key and value side by side."""
    buf = torch.zeros(shape, dtype=BF16)
    buf = buf if order is None else buf.permute(order)
    if buf.ndim == 4:
        q, k, v = buf.split([4, 2, 2], at)
    else:
        q, k, v = buf.unbind(at)
    assert q.shape[:2] == (2, 3)
    for x, y, z in ((q, k, v), (q, v, k)) + (((k, q, v), (v, k, q)) if buf.ndim == 5 else ()):
        with pytest.raises(ValueError, match="runs on a ROCm GPU"):
            call(q=x, out=x, k=y, v=z)
        with pytest.raises(ValueError, match="k and v must lie apart"):
            call(q=x, out=x, k=y, v=x[:, :, :2])


def test_apart_sees_every_order_of_a_projection():
    """Of random slices of one tensor in any order of its dimensions: the same as
    by their elements."""
    gen = torch.Generator().manual_seed(1)
    seen = {True: 0, False: 0}
    for _ in range(3000):
        N, T, H, third = (int(x) for x in torch.randint(1, 4, (4,), generator=gen))
        order = torch.randperm(4, generator=gen).tolist()
        buf = torch.arange(N * T * H * third * 2).view(*[(N, T, H, third)[i] for i in order], 2)
        buf = buf.permute(*[order.index(i) for i in range(4)], 4)
        if third > 1:
            a, b = (buf[:, :, :, int(i)] for i in torch.randint(third, (2,), generator=gen))
        else:
            (i, j), (k, l) = (sorted(torch.randint(H, (2,), generator=gen).tolist()) for _ in range(2))
            a, b = buf[:, :, i:j + 1, 0], buf[:, :, k:l + 1, 0]
        common = bool(set(a.flatten().tolist()) & set(b.flatten().tolist()))
        assert _apart(a, b) != common, (a.shape, a.stride(), b.shape, b.stride(), a.storage_offset(), b.storage_offset())
        seen[common] += 1
    assert min(seen.values()) > 500, seen


def test_apart_means_no_element_in_common():
    gen = torch.Generator().manual_seed(0)

    def draw(*choices):
        return choices[int(torch.randint(len(choices), (1,), generator=gen))]

    buf, seen = torch.arange(600), {True: 0, False: 0}
    for _ in range(4000):
        N, T = draw(1, 2, 3), draw(1, 2, 3)
        rows, tokens = draw(12, 24, 30, 36, 72), draw(4, 8, 10, 12, 24)
        a, b = (buf.as_strided((N, T, draw(1, 2), 2), (draw(rows, rows, rows, 18), draw(tokens, tokens, tokens, 6), draw(2, 4, 12), 1),
                               draw(0, 2, 4, 6, 8, 12, 36, 72, 200)) for _ in range(2))
        apart = _apart(a, b)
        assert not apart or not set(a.flatten().tolist()) & set(b.flatten().tolist()), (a.shape, a.stride(), b.shape, b.stride())
        seen[apart] += 1
    assert min(seen.values()) > 400, seen


@pytest.mark.parametrize("name", ["q", "k", "v", "k_cache", "v_cache", "inv_freq", "out"])
def test_a_gradient_is_refused(name):
    shapes = dict(q=(2, 3, 4, 64), k=(2, 3, 2, 64), v=(2, 3, 2, 64), k_cache=(5, 16, 2, 64), v_cache=(5, 16, 2, 64),
                  inv_freq=(32,), out=(2, 3, 4, 64))
    t = torch.zeros(shapes[name], dtype=torch.float32 if name == "inv_freq" else BF16, requires_grad=True)
    with pytest.raises(NotImplementedError, match="paged_append_rotary is forward only: inputs require grad"):
        call(**{name: t})
    with torch.no_grad(), pytest.raises(ValueError, match="runs on a ROCm GPU"):
        call(**{name: t})


def test_struct_matches_the_header():
    cls = _hip.KdaPagedRotaryArgs
    body = re.search(r"typedef struct KdaPagedRotaryArgs \{(.*?)\} KdaPagedRotaryArgs;", _text(), re.S).group(1)
    names = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        names += [n.strip().lstrip("*") for n in re.sub(r"^.*?\b(?=\w+\s*(,|$))", "", decl).split(",")]
    assert names == [f for f, _ in cls._fields_]


@pytest.mark.skipif(shutil.which("gcc") is None, reason="no C compiler")
def test_c_compiler_sees_the_same_layout(tmp_path):
    cls = _hip.KdaPagedRotaryArgs
    lines = ['printf("%zu\\n", sizeof(KdaPagedRotaryArgs));']
    lines += [f'printf("%zu\\n", offsetof(KdaPagedRotaryArgs, {f}));' for f, _ in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "kda_paged_hip.h"\nint main(void) {\n'
                   + "\n".join(lines) + "\nreturn 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", f"-I{HEADER.parent}", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()
    assert [int(x) for x in out] == [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_]


def test_packed_arguments_are_the_struct():
    base = paged()
    tail = dict(inv_freq=11, rotary_dim=64, interleaved=1, q_out=12, out_row=13, out_token=14, out_head=15)
    flat = [getattr(base, f) or 0 for f, _ in base._fields_]
    assert _hip.PAGED_ROTARY_PACK.pack(*flat, *tail.values()) == bytes(_hip.KdaPagedRotaryArgs(base, *tail.values()))


def rotary(base=None, **change):
    tail = dict(inv_freq=FAKE, rotary_dim=128, interleaved=0, q_out=FAKE, out_row=512, out_token=512, out_head=128) | change
    return _hip.KdaPagedRotaryArgs(paged(**(base or {})), *tail.values())


@fake_pointers
def test_argument_checks():
    f = _hip.lib().kda_paged_append_rotary_hip
    assert f(None, None) == -1
    assert f(ctypes.byref(rotary(dict(abi_version=99))), None) == -5
    for bad in (dict(HQ=0), dict(q=0), dict(q=FAKE + 8), dict(q_head=4), dict(q_token=-8), dict(new_k=0), dict(nv_head=4),
                dict(page_table=0), dict(N=0), dict(k=FAKE + 8)):
        assert f(ctypes.byref(rotary(bad)), None) == -1, bad
    for bad in (dict(inv_freq=0), dict(inv_freq=FAKE + 2), dict(q_out=0), dict(q_out=FAKE + 8), dict(out_head=4),
                dict(out_row=-8)):
        assert f(ctypes.byref(rotary(**bad)), None) == -1, bad
    for bad in (dict(rotary_dim=0), dict(rotary_dim=8), dict(rotary_dim=24), dict(rotary_dim=144)):
        assert f(ctypes.byref(rotary(**bad)), None) == -2, bad
    assert f(ctypes.byref(rotary(dict(D=96))), None) == -2
    # threads past 32 bits
    assert f(ctypes.byref(rotary(dict(N=1 << 20, T=1 << 6, HQ=1))), None) == -2
    assert f(ctypes.byref(rotary(dict(HQ=(1 << 31) - 1))), None) == -2
