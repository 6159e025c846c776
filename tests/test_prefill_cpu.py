"""Argument checks of prefill_attention without a GPU."""

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
    lib.pkv_prefill_attention.argtypes = [P, P, P, I, P, P, P, P, I, L, L, I, I, I, L, L, L, L, L, L,
                                          ct.c_float, I, P]
    return lib


FULL = dict(q=16, k=16, v=16, out=16, cq=16, ck=16)


def call(lib, **kw):
    a = dict(q=None, k=None, v=None, dtype=2, out=None, lse=None, cq=None, ck=None, seqs=2, tq=10,
             tk=10, heads=8, kv=2, dim=128, qt=1024, qh=128, kt=256, kh=128, vt=256, vh=128,
             scale=0.1, causal=1)
    a.update(kw)
    return lib.pkv_prefill_attention(*a.values(), None)


@pytest.mark.parametrize("kw,rc,msg", [
    (dict(dtype=0), 1, "float16"), (dict(dtype=3), 1, "float16"), (dict(dim=132), 1, "head_dim"),
    (dict(dim=136), 1, "head_dim"), (dict(dim=0), 1, "head_dim"), (dict(kv=3), 1, "GQA"),
    (dict(kv=0), 1, "shape"), (dict(seqs=-1), 1, "shape"), (dict(heads=129, kv=1), 2, "128"),
    (dict(scale=0.0), 1, "sm_scale"), (dict(scale=-1.0), 1, "sm_scale"),
    (dict(scale=float("inf")), 1, "sm_scale"), (dict(scale=float("nan")), 1, "sm_scale"),
    (dict(), 1, "null"), (dict(FULL, qt=1028), 1, "strides"), (dict(FULL, vh=0), 1, "strides"),
    (dict(FULL, k=24), 1, "aligned"), (dict(FULL, tq=1 << 31), 2, "rows"),
])
def test_refuses(lib, kw, rc, msg):
    assert call(lib, **kw) == rc
    assert re.search(msg, lib.pkv_last_error_string().decode())


def test_nothing_to_do_is_ok(lib):
    assert call(lib, tq=0) == 0


def test_host_tensors_need_a_device():
    from pagedkv_fusion import _C
    x = torch.zeros(1, 2, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        _C.prefill_attention(x, x, x, torch.zeros(2, dtype=torch.int32), 0.1)
