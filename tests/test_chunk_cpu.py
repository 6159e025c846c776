"""Argument checks of chunk_attention, accumulate_attention and evict_tokens without a GPU."""

from __future__ import annotations

import ctypes as ct
import re

import pytest
import torch

from conftest import ensure_native_built

P, I, L, F, Z = ct.c_void_p, ct.c_int32, ct.c_int64, ct.c_float, ct.c_size_t


@pytest.fixture(scope="module")
def lib():
    lib = ct.CDLL(str(ensure_native_built()))
    lib.pkv_last_error_string.restype = ct.c_char_p
    lib.pkv_chunk_attention.argtypes = [P, I] + [P] * 9 + [L] + [I] * 5 + [L, I, L, L, F, P, Z, P]
    lib.pkv_accumulate_attention.argtypes = [P, P, I] + [P] * 6 + [L] + [I] * 5 + [L, I, L, L, F, P, Z, P]
    lib.pkv_evict_tokens.argtypes = [P] * 7 + [I, L] + [I] * 7 + [P]
    for name, args in (("chunk_attention", [L] + [I] * 6),
                       ("accumulate_attention", [L] + [I] * 5 + [L, I, I])):
        f = getattr(lib, f"pkv_{name}_workspace_size")
        f.argtypes, f.restype = args, Z
    return lib


SIZES = dict(T=20, S=4, H=8, Hkv=2, D=128, bs=16, NB=100, M=8, qt=1024, qh=128)


def chunk(lib, ptrs, dtype=1, **kw):
    a = dict(SIZES, **kw)
    return lib.pkv_chunk_attention(ptrs[0], dtype, *ptrs[1:], *a.values(), 0.1, None, 0, None)


def accumulate(lib, ptrs, dtype=1, **kw):
    a = dict(SIZES, **kw)
    return lib.pkv_accumulate_attention(*ptrs[:2], dtype, *ptrs[2:], *a.values(), 0.1, None, 0, None)


COMMON = [
    (dict(D=48), 1, "head_dim"), (dict(D=288), 1, "head_dim"), (dict(bs=65), 1, "block_size"),
    (dict(bs=0), 1, "block_size"), (dict(Hkv=3), 1, "multiple of num_kv_heads"), (dict(Hkv=0), 1, "shape"),
    (dict(T=-1), 1, "shape"), (dict(dtype=3), 1, "float32"), (dict(qt=1020), 1, "strides"),
    (dict(qh=130), 1, "strides"), (dict(dtype=0, qt=1022), 1, "strides"), (dict(T=1 << 29), 2, "2\\^31"),
    (dict(M=1 << 28), 2, "2\\^31"), (dict(NB=1 << 28), 2, "2\\^31"), ({}, 3, "workspace"),
]


@pytest.mark.parametrize("kw,rc,msg", COMMON)
def test_refuses(lib, kw, rc, msg):
    kw = dict(kw)
    dtype = kw.pop("dtype", 1)
    assert chunk(lib, [16] * 10, dtype, **kw) == rc
    assert re.search(msg, lib.pkv_last_error_string().decode())
    assert accumulate(lib, [16] * 8, dtype, **kw) == rc
    assert re.search(msg, lib.pkv_last_error_string().decode())


@pytest.mark.parametrize("missing", range(9))
def test_refuses_null_pointers(lib, missing):
    ptrs = [16] * 10
    ptrs[missing] = None  # (9 is lse, which may be missing)
    assert chunk(lib, ptrs) == 1 and b"null" in lib.pkv_last_error_string()
    if missing < 7:
        ptrs = [16] * 8
        ptrs[missing] = None
        assert accumulate(lib, ptrs) == 1 and b"null" in lib.pkv_last_error_string()


def test_refuses_addresses_and_too_many_rows(lib):
    for at in (0, 1, 3, 8):
        ptrs = [16] * 10
        ptrs[at] = 24
        assert chunk(lib, ptrs) == 1 and b"aligned" in lib.pkv_last_error_string()
    assert accumulate(lib, [16] * 8, T=(1 << 22) + 1) == 2
    assert b"2^25" in lib.pkv_last_error_string()


def test_nothing_to_do_is_ok(lib):
    assert chunk(lib, [None] * 10, T=0) == 0
    assert accumulate(lib, [None] * 8, T=0) == 0
    assert accumulate(lib, [16] * 8, M=0) == 0
    assert evict(lib, [None] * 7, S=0) == 0


def evict(lib, ptrs, **kw):
    a = dict(S=4, NB=100, bs=16, Hkv=2, D=64, M=8, keep=10, sinks=2, recent=3)
    a.update(kw)
    return lib.pkv_evict_tokens(*ptrs, *a.values(), None)


@pytest.mark.parametrize("kw,rc,msg", [
    (dict(keep=0, sinks=0, recent=0), 1, "keep"), (dict(sinks=-1), 1, "keep"), (dict(recent=-1), 1, "keep"),
    (dict(sinks=8), 1, "keep"), (dict(D=257), 1, "head_dim"), (dict(bs=65), 1, "block_size"),
    (dict(Hkv=0), 1, "shape"), (dict(NB=1 << 28), 2, "2\\^31"), (dict(M=1 << 28), 2, "2\\^31"),
    (dict(S=1 << 27), 2, "CTAs"),
])
def test_evict_refuses(lib, kw, rc, msg):
    assert evict(lib, [16] * 7, **kw) == rc
    assert re.search(msg, lib.pkv_last_error_string().decode())


@pytest.mark.parametrize("missing", range(7))
def test_evict_refuses_null_pointers(lib, missing):
    ptrs = [16] * 7
    ptrs[missing] = None
    assert evict(lib, ptrs) == 1 and b"null" in lib.pkv_last_error_string()


def test_workspaces(lib):
    f, g = lib.pkv_chunk_attention_workspace_size, lib.pkv_accumulate_attention_workspace_size
    assert f(0, 4, 32, 8, 128, 16, 100) == 0 and f(64, 64, 32, 8, 48, 16, 100) == 0
    # two parts a warp of the grid, whatever the lengths
    assert f(64, 64, 32, 8, 128, 16, 100) == f(64, 64, 32, 8, 128, 16, 10000) < 32 << 20
    # sums of one word a cache slot; without lse the scores of a decode step too
    words = 1000 * 16 * 8
    given, first = g(64, 64, 32, 8, 128, 16, 1000, 10, 1), g(64, 64, 32, 8, 128, 16, 1000, 10, 0)
    assert words <= given < words + 8192 and first >= given + 64 * 32 * 4 * (1 + 160)
    assert g(64, 64, 32, 8, 128, 16, 1000, 0, 0) == 0
    # scores of at most 128 MB: above that the pass is repeated
    assert g(64, 64, 32, 8, 128, 16, 1000, 1 << 20, 0) < 256 << 20


def test_host_tensors_need_a_device():
    from pagedkv_fusion import _C
    x = torch.zeros(1, 2, 64)
    for call in (lambda: _C.chunk_attention(x, *([x] * 7), 0.1),
                 lambda: _C.accumulate_attention(x, *([x] * 6), 0.1),
                 lambda: _C.evict_tokens(*([x] * 5), 4)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
