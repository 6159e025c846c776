"""prefill_attention's workspace for long key ranges, without a GPU."""

from __future__ import annotations

import ctypes as ct

import pytest

from test_prefill_cpu import FULL, I, L, P, lib  # noqa: F401


@pytest.fixture(scope="module")
def entry(lib):  # noqa: F811
    lib.pkv_prefill_attention_workspace_size.argtypes = [L, L, I]
    lib.pkv_prefill_attention_workspace_size.restype = ct.c_size_t
    lib.pkv_prefill_attention_ws.argtypes = lib.pkv_prefill_attention.argtypes[:-1] + [P, ct.c_size_t, P]
    return lib


def test_size(entry):
    size = entry.pkv_prefill_attention_workspace_size
    assert size(10, 16384, 128) == 0 and size(10, 1 << 30, 64) == 0 and size(0, 1 << 30, 128) == 0
    assert size(10, 16385, 128) == size(1 << 20, 1 << 30, 72) >= 148 * 2 * 128 * 128 * 4


def test_too_small_a_workspace_is_refused(entry):
    a = dict(q=None, k=None, v=None, dtype=2, out=None, lse=None, cq=None, ck=None, seqs=2, tq=10,
             tk=20000, heads=8, kv=2, dim=128, qt=1024, qh=128, kt=256, kh=128, vt=256, vh=128,
             scale=0.1, causal=1)
    a.update(FULL)
    assert entry.pkv_prefill_attention_ws(*a.values(), 4096, 1000, None) == 3
    assert b"workspace" in entry.pkv_last_error_string()
    a.update(dim=132)   # the checks of the call without one
    assert entry.pkv_prefill_attention_ws(*a.values(), 4096, 1 << 30, None) == 1
    a.update(dim=128, tq=0)
    assert entry.pkv_prefill_attention_ws(*a.values(), None, 0, None) == 0
