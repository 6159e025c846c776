"""Argument checks of shared_prefix_attention without a GPU."""

from __future__ import annotations

import ctypes as ct
import re

import pytest
import torch

from conftest import ensure_native_built

P, I, L = ct.c_void_p, ct.c_int32, ct.c_int64


@pytest.fixture(scope="module")
def lib():
    lib = ct.CDLL(str(ensure_native_built()))
    lib.pkv_last_error_string.restype = ct.c_char_p
    lib.pkv_shared_prefix_attention.argtypes = [P] * 10 + [I] * 5 + [L, I, I, ct.c_float, P,
                                                                     ct.c_size_t, P]
    f = lib.pkv_shared_prefix_attention_workspace_size
    f.argtypes = [I] * 5 + [L, I, I]
    f.restype = ct.c_size_t
    return lib


def call(lib, ptr=None, **kw):
    a = dict(S=4, H=8, Hkv=2, D=128, bs=16, NB=100, P=32, M=8)
    a.update(kw)
    ptrs = list(ptr) if ptr else [None] * 10
    return lib.pkv_shared_prefix_attention(*ptrs, *a.values(), 0.1, None, 0, None)


@pytest.mark.parametrize("ptr,kw,rc,msg", [
    (None, dict(D=48), 1, "head_dim"), (None, dict(D=160), 1, "null|head_dim"),
    ([16] * 10, dict(D=160), 1, "head_dim"), (None, dict(bs=65), 1, "block_size"),
    (None, dict(Hkv=3), 1, "GQA"), (None, {}, 1, "null"),
    ([16] * 5 + [None] + [16] * 4, {}, 1, "null"), ([16] * 6 + [None] + [16] * 3, {}, 1, "null"),
    ([16] * 10, dict(P=-1), 1, "prefix"), ([20] + [16] * 9, {}, 1, "aligned"),
    ([16] * 10, dict(P=1 << 30), 2, "2\\^31"), ([16] * 10, {}, 3, "workspace"),
])
def test_refuses(lib, ptr, kw, rc, msg):
    assert call(lib, ptr, **kw) == rc
    assert re.search(msg, lib.pkv_last_error_string().decode())


def test_nothing_to_do_is_ok(lib):
    assert call(lib, S=0) == 0


def test_workspace_holds_both_parts(lib):
    f = lib.pkv_shared_prefix_attention_workspace_size
    rows = 64 * 32
    none, pre = f(64, 32, 8, 128, 16, 1000, 0, 0), f(64, 32, 8, 128, 16, 1000, 128, 0)
    both = f(64, 32, 8, 128, 16, 1000, 128, 32)
    assert none < 4096 and pre >= rows * 128 * 4 and both >= pre + rows * 128 * 4
    assert f(0, 32, 8, 128, 16, 1000, 128, 32) == 0
    # the prefix is split over at most one CTA per SM and tile
    assert f(1, 8, 8, 128, 16, 1 << 20, 1 << 19, 0) <= 148 * 8 * (128 * 4 + 8) + 4096


def test_host_tensors_need_a_device():
    from pagedkv_fusion import _C
    x = torch.zeros(1, 2, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        _C.shared_prefix_attention(x, *([x] * 8), 0.1)
