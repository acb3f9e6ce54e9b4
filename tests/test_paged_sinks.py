"""First tokens that stay visible: checks of arguments and the C ABI (CPU only)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from kda_bt16 import _hip
from test_paged_capi import FAKE, fake_pointers, paged
from test_paged_validation import attention


def test_refusals():
    for kw, match in ((dict(sinks=-1, window=4), "sinks must not be negative, got -1"), (dict(sinks=4), "sinks needs a window"),
                      (dict(sinks=4, causal=False), "sinks needs a window"),
                      (dict(sinks=4, window=0), "window must be at least 1"),
                      (dict(sinks=4, window=2, causal=False), "window needs causal")):
        with pytest.raises(ValueError, match=match):
            attention(**kw)
    with pytest.raises(ValueError, match="runs on a ROCm GPU"):
        attention(sinks=4, window=10)
    with pytest.raises(NotImplementedError, match="forward only"):
        attention(sinks=4, window=10, q=torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16, requires_grad=True))


def sinks(n, **base):
    return _hip.KdaPagedSinksArgs(paged(**dict(flags=_hip.PAGED_CAUSAL, window=100) | base), n, 0)


def test_struct_and_packing():
    a = sinks(7)
    assert ctypes.sizeof(a) == ctypes.sizeof(_hip.KdaPagedArgs) + 8
    assert bytes(a) == bytes(a.paged) + _hip.SINKS_PACK.pack(7, 0)


def test_workspace_follows_what_can_be_seen():
    f, plain = _hip.lib().kda_paged_attn_sinks_workspace_bytes, _hip.lib().kda_paged_attn_workspace_bytes
    few = 2 * 512 * 32 * 130 * 4
    assert f(None) == 0
    # 768 keys in whole tiles: one launch, however wide the table is
    for w, s, want in ((100, 4, 0), (608, 32, 0), (609, 32, few), (5000, 4, few), (100, 5000, few)):
        assert f(ctypes.byref(sinks(s, window=w, M=1000, table_stride=1000))) == want, (w, s)
    assert f(ctypes.byref(sinks(5000, window=5000, M=48, table_stride=48))) == 0  # (no more keys than the table)
    assert plain(ctypes.byref(paged(M=1000, table_stride=1000))) == few


@fake_pointers
def test_argument_checks():
    f = _hip.lib().kda_paged_attn_sinks_hip
    assert f(None, None) == -1
    assert f(ctypes.byref(sinks(-1)), None) == -1
    assert f(ctypes.byref(sinks(4, window=0)), None) == -2  # every key is visible
    assert f(ctypes.byref(sinks(4, flags=0)), None) == -2
    assert f(ctypes.byref(sinks(4, abi_version=9)), None) == -5
    assert f(ctypes.byref(sinks(4, q=0)), None) == -1 and f(ctypes.byref(sinks(4, D=96)), None) == -2
    big = dict(window=5000, M=1000, table_stride=1000)
    assert f(ctypes.byref(sinks(4, **big)), None) == -3  # no workspace
    assert f(ctypes.byref(sinks(4, workspace=FAKE + 16, workspace_bytes=1 << 30, **big)), None) == -3
