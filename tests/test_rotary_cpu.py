"""Argument checks of qk_norm_rope and append_kv and the rotary table, without
a GPU: the C entry points refuse before they touch the device."""

from __future__ import annotations

import ctypes as ct

import numpy as np
import pytest
import torch

from conftest import ensure_native_built

P, I, L = ct.c_void_p, ct.c_int32, ct.c_int64


@pytest.fixture(scope="module")
def lib():
    lib = ct.CDLL(str(ensure_native_built()))
    lib.pkv_last_error_string.restype = ct.c_char_p
    lib.pkv_qk_norm_rope.argtypes = [P, P, I, P, P, P, P, P, P, I, ct.c_float, L, I, I, I, I, L, I,
                                     L, L, L, L, P]
    lib.pkv_append_kv.argtypes = [P, P, I, P, P, P, P, P, L, L, I, I, I, I, L, I, L, L, L, L, P,
                                  ct.c_size_t, P]
    lib.pkv_append_kv_workspace_size.argtypes = [L, L]
    lib.pkv_append_kv_workspace_size.restype = ct.c_size_t
    return lib


def rope(lib, **kw):
    a = dict(q=None, k=None, dtype=1, qo=None, ko=None, pos=None, table=None, qw=None, kw=None,
             wf=0, eps=1e-6, tokens=4, heads=8, kv=2, dim=128, rot=128, n=16, inter=0)
    a.update(kw)
    return lib.pkv_qk_norm_rope(*a.values(), 1024, 128, 256, 128, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=3), "float32"), (dict(tokens=-1), "shape"), (dict(dim=257), "head_dim"),
    (dict(dim=0), "head_dim"), (dict(rot=130), "rotary_dim"), (dict(rot=63), "rotary_dim"),
    (dict(), "null"), (dict(n=-1), "num_positions"),
    (dict(q=16, k=16, qo=16, ko=16, pos=16, table=16, qw=16), "go together"),
    (dict(q=16, k=16, qo=16, ko=16, pos=16, table=16, tokens=1 << 29), "2\\^31"),
])
def test_qk_norm_rope_refuses(lib, kw, msg):
    assert rope(lib, **kw) in (1, 2)
    import re
    assert re.search(msg, lib.pkv_last_error_string().decode())


def append(lib, **kw):
    a = dict(k=None, v=None, dtype=1, cache=None, scales=None, slots=None, pos=None, table=None,
             tokens=4, blocks=8, bs=16, kv=2, dim=128, rot=0, n=0, inter=0)
    a.update(kw)
    return lib.pkv_append_kv(*a.values(), 256, 128, 256, 128, None, 0, None)


FULL = dict(k=16, v=16, cache=16, scales=16, slots=16)


@pytest.mark.parametrize("kw,rc,msg", [
    (dict(dtype=-1), 1, "float32"), (dict(bs=65), 1, "block_size"), (dict(bs=0), 1, "block_size"),
    (dict(dim=260), 1, "head_dim"), (dict(kv=0), 1, "shape"), (dict(), 1, "null"),
    (dict(FULL, pos=16), 1, "go together"),
    (dict(FULL, pos=16, table=16, rot=129, n=4), 1, "rotary_dim"),
    (dict(FULL, tokens=1 << 31), 2, "2\\^31"),
    (dict(FULL, tokens=5000), 3, "workspace"),
])
def test_append_kv_refuses(lib, kw, rc, msg):
    import re
    assert append(lib, **kw) == rc
    assert re.search(msg, lib.pkv_last_error_string().decode())


def test_nothing_to_do_is_ok(lib):
    assert rope(lib, tokens=0) == 0
    assert append(lib, tokens=0) == 0


def test_append_workspace_grows_with_the_call(lib):
    assert lib.pkv_append_kv_workspace_size(1, 1000) == 0
    assert lib.pkv_append_kv_workspace_size(5000, 1000) >= 4 * (1000 + 2 * 5000)
    assert lib.pkv_append_kv_workspace_size(0, 1000) == 0


def test_host_tensors_are_refused_by_the_append():
    from pagedkv_fusion import _C
    x = torch.zeros(1, 2, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        _C.append_kv(x, x, torch.zeros(2, 1, 16, 2, 64, dtype=torch.int8), torch.ones(2, 1, 2),
                     torch.zeros(1, dtype=torch.int64), 16)


def test_rotary_table_on_the_host():
    from pagedkv_fusion import ops
    t = ops.rotary_table(300001, 64, base=500000.0, device="cpu")
    f = 500000.0 ** (-np.arange(0, 64, 2) / 64)
    at = np.array([0, 17, 300000])
    want = np.concatenate([np.cos(at[:, None] * f), np.sin(at[:, None] * f)], 1)
    assert t.dtype == torch.float32 and t.shape == (300001, 64)
    # float32 rounding of values up to 1, and the angle's rounding in 64 bits
    assert np.abs(t.numpy()[at] - want).max() <= 2.0 ** -25 + 1e-9
    far = ops.rotary_table(8, 64, scaling="ntk", factor=4.0, device="cpu").numpy()
    near = ops.rotary_table(8, 64, device="cpu").numpy()
    np.testing.assert_array_equal(far[:, 0], near[:, 0])   # the fastest pair is kept
    slow = lambda t: np.arctan2(t[1, 63], t[1, 31])         # noqa: E731
    np.testing.assert_allclose(slow(far), slow(near) / 4, rtol=1e-5)
