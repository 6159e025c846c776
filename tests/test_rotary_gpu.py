"""qk_norm_rope and append_kv against plain 64-bit implementations.

Tolerances: qk_norm_rope computes in 32 bits and rounds once, so an output is
off by half a step of its type (``finfo(t).eps / 2`` of the value) plus the
32-bit arithmetic: a sum of up to 256 squares, one rsqrt, four products and a
sum, under 2^-24 * (256 + 8) of the pair's length in the worst case.  append_kv
has one defined value per code and scale: they must be equal to the same
steps taken in numpy float32.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def rotate64(x, rows, interleaved):
    """x [T, H, D] float64, rows [T, R] float64."""
    r = rows.shape[1]
    c, s = rows[:, None, :r // 2], rows[:, None, r // 2:]
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y[..., 0:r:2], y[..., 1:r:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        y[..., :r // 2], y[..., r // 2:r] = a * c - b * s, b * c + a * s
    return y


def expected_qk(x, positions, table, weight, eps, interleaved):
    y = x.double()
    if weight is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    return rotate64(y, table.double()[positions], interleaved)


def assert_rope_close(got, want, dtype):
    length = want.abs().amax(-1, keepdim=True)  # bounds either member of a pair within sqrt(2)
    tol = torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -24 * 264 * 1.5 * length + 1e-30
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25  # half a step of its subnormals
    assert got.dtype == dtype
    assert bool(((got.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rot,interleaved,norm", [
    (1, 8, 8, 128, 128, False, True),
    (64, 32, 8, 128, 128, False, True),
    (700, 12, 4, 128, 64, True, False),
    (33, 6, 2, 64, 32, False, True),
    (5, 3, 1, 80, 20, True, True),
    (5, 3, 1, 80, 20, False, False),    # R/2 = 10: the scalar kernel
    (300, 40, 40, 96, 96, False, False),
    (17, 2, 1, 256, 256, False, True),
    (17, 2, 1, 256, 64, True, True),
    (9, 14, 2, 32, 8, False, True),
    (9, 5, 1, 33, 32, False, True),     # odd head dim
    (9, 5, 1, 33, 0, False, True),      # nothing rotated
    (2500, 32, 8, 128, 128, True, True),
])
def test_qk_norm_rope(cuda, dtype, tokens, heads, kv_heads, dim, rot, interleaved, norm):
    from pagedkv_fusion import ops
    dt = DTYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(tokens + dim)
    qkv = torch.randn(tokens, heads + 2 * kv_heads, dim, generator=g, device="cuda").to(dt)
    q, k = qkv[:, :heads], qkv[:, heads:heads + kv_heads]
    table = ops.rotary_table(4096, rot)
    pos = torch.randint(4096, (tokens,), generator=g, device="cuda")
    qw = kw = None
    if norm:
        qw, kw = (1 + 0.2 * torch.randn(2, dim, generator=g, device="cuda")).to(dt)
    qo, ko = ops.qk_norm_rope(q, k, pos, table, qw, kw, 1e-5, interleaved)
    assert qo.is_contiguous() and ko.is_contiguous()
    assert_rope_close(qo, expected_qk(q, pos, table, qw, 1e-5, interleaved), dt)
    assert_rope_close(ko, expected_qk(k, pos, table, kw, 1e-5, interleaved), dt)
    if norm:  # float32 weights
        qo, ko = ops.qk_norm_rope(q, k, pos.int(), table, qw.float(), kw.float(), 1e-5, interleaved)
        assert_rope_close(ko, expected_qk(k, pos, table, kw, 1e-5, interleaved), dt)
    qo, none = ops.qk_norm_rope(q, None, pos, table, interleaved=interleaved)
    assert none is None
    assert_rope_close(qo, expected_qk(q, pos, table, None, 0.0, interleaved), dt)
    assert cuda.read_device_error() == 0


def test_qk_norm_rope_strides_and_alignment(cuda):
    from pagedkv_fusion import ops
    g = torch.Generator(device="cuda").manual_seed(3)
    base = torch.randn(50 * 9 * 130 + 1, generator=g, device="cuda").half()
    table = ops.rotary_table(64, 128)
    pos = torch.arange(50, device="cuda")
    odd = base[1:].view(50, 9, 130)[..., :128]                 # misaligned, padded rows
    swapped = base[:50 * 9 * 128].view(9, 50, 128).transpose(0, 1)
    columns = base[:50 * 9 * 128].view(50, 128, 9).transpose(1, 2)  # channels not contiguous
    same = swapped[:, :1].expand(50, 9, 128)                   # stride 0
    for q in (odd, swapped, columns, same):
        k = q[:, :2]
        qo, ko = ops.qk_norm_rope(q, k, pos, table)
        assert_rope_close(qo, expected_qk(q, pos, table, None, 0, False), torch.float16)
        assert_rope_close(ko, expected_qk(k, pos, table, None, 0, False), torch.float16)


def test_qk_norm_rope_values_outside_the_rotation_stay(cuda):
    """Infinities and NaN in channels that are not rotated reach no others,
    and a token with a bad position is zero and reported."""
    from pagedkv_fusion import ops
    q = torch.randn(6, 4, 128, device="cuda").bfloat16()
    q[0, :, 100] = float("inf")
    q[1, :, 101] = float("nan")
    table = ops.rotary_table(16, 36)  # ends inside a 16-byte chunk
    pos = torch.tensor([0, 3, 16, 5, -1, 15], device="cuda")
    for interleaved in (False, True):
        out, _ = ops.qk_norm_rope(q, None, pos, table, interleaved=interleaved)
        assert cuda.read_device_error() == 5
        assert bool((out[2] == 0).all()) and bool((out[4] == 0).all())
        good = [0, 1, 3, 5]
        want = expected_qk(q[good], pos[good], table, None, 0, interleaved)
        ok = want.isfinite()
        assert torch.equal(out[good].isfinite(), ok)
        assert torch.equal(out[good][..., 36:].nan_to_num(7), q[good][..., 36:].nan_to_num(7))
        assert int((~ok).sum()) == 8


@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "yarn"])
def test_rotary_table(cuda, scaling):
    from pagedkv_fusion import ops
    r, n, base, factor, orig = 128, 200000, 10000.0, 8.0, 4096
    t = ops.rotary_table(n, r, base, scaling, factor, orig)
    i = np.arange(64, dtype=np.float64)
    f, mag = base ** (-2 * i / r), 1.0
    if scaling == "linear":
        f = f / factor
    if scaling == "ntk":
        f = (base * factor ** (128 / 126)) ** (-2 * i / r)
    if scaling == "yarn":
        turns = orig * f / (2 * np.pi)  # falls with the pair
        assert np.all(np.diff(turns) < 0)
        kept = ops.rotary_table(2, r, base, "none").double().cpu().numpy()
        one = t[1].double().cpu().numpy() / (0.1 * np.log(factor) + 1)
        got = np.arctan2(one[64:], one[:64])
        np.testing.assert_allclose(got[turns > 40], np.arctan2(kept[1, 64:], kept[1, :64])[turns > 40],
                                   rtol=1e-6)
        np.testing.assert_allclose(got[turns < 0.7], f[turns < 0.7] / factor, rtol=1e-6)
        between = (turns < 32) & (turns > 1)
        assert np.all(got[between] <= f[between] * (1 + 1e-6))
        assert np.all(got[between] >= f[between] / factor * (1 - 1e-6))
        return
    at = np.array([0, 1, 4095, 131071, n - 1])
    want = np.concatenate([np.cos(at[:, None] * f), np.sin(at[:, None] * f)], 1) * mag
    # float32 rounding of values up to 1, and the angle's own 64-bit rounding (2e5 * 2^-52)
    assert np.abs(t.cpu().numpy()[at] - want).max() <= 2.0 ** -25 + 1e-9


# ---------------------------------------------------------------------------
# append_kv
# ---------------------------------------------------------------------------

def np_rotate32(x, rows, interleaved):
    r = rows.shape[1]
    c, s = rows[:, None, :r // 2], rows[:, None, r // 2:]
    y = x.copy()
    if interleaved:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y[..., 0:r:2], y[..., 1:r:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        y[..., :r // 2], y[..., r // 2:r] = a * c - b * s, b * c + a * s
    return y


def np_append(key, value, cache, scales, slots, bs, rows=None, interleaved=False):
    """The definition, page by page, each float32 step rounded by numpy."""
    nb = cache.shape[1]
    if rows is not None:
        key = np_rotate32(key, rows, interleaved)
    pages = {}
    for t, s in enumerate(slots):
        if 0 <= s < nb * bs:
            pages.setdefault(int(s) // bs, {})[int(s) % bs] = t  # the last token of a slot
    for page, toks in pages.items():
        lowest = min(toks)
        for plane, x in ((0, key), (1, value)):
            new = x[list(toks.values())]                       # [n, Hkv, D]
            amax = np.abs(new).max((0, 2)).astype(np.float32)  # NaN wins
            with np.errstate(invalid="ignore"):
                step = np.where(amax > 0, amax / np.float32(127), np.float32(0)).astype(np.float32)
            old = scales[plane, page].copy()
            sc = np.where(step > 0, step, np.float32(1)) if lowest == 0 else np.where(step > old, step, old)
            if lowest > 0:
                for h in np.nonzero(step > old)[0]:
                    ratio = np.float32(old[h] / sc[h])
                    c = cache[plane, page, :lowest, h].astype(np.float32)
                    cache[plane, page, :lowest, h] = np.rint(c * ratio).astype(np.int8)
            scales[plane, page] = sc
            for off, t in toks.items():
                with np.errstate(invalid="ignore", divide="ignore"):
                    q = np.rint((x[t] / sc[:, None]).astype(np.float32))
                cache[plane, page, off] = np.clip(np.nan_to_num(q, nan=-127), -127, 127).astype(np.int8)


def check_append(cuda, key, value, cache, scales, slots, bs, positions=None, table=None,
                 interleaved=False, error=0):
    from pagedkv_fusion import ops
    c, s = cache.cpu().numpy().copy(), scales.cpu().numpy().copy()
    rows = None if table is None else table.cpu().numpy()[positions.clamp(0, len(table) - 1).cpu().numpy()]
    np_append(key.float().cpu().numpy(), value.float().cpu().numpy(), c, s, slots.cpu().numpy(), bs,
              rows, interleaved)
    ops.append_kv(key, value, cache, scales, slots, bs, positions, table, interleaved)
    assert cuda.read_device_error() == error
    np.testing.assert_array_equal(scales.cpu().numpy().view(np.uint32), s.view(np.uint32))
    np.testing.assert_array_equal(cache.cpu().numpy(), c)


def append_problem(seed, counts, fills, kv_heads, dim, bs, dtype, rot):
    from pagedkv_fusion import ops
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = [-(-(f + c) // bs) for f, c in zip(fills, counts)]
    nb = sum(pages) + 2
    perm = torch.randperm(nb, generator=g, device="cuda").cpu().numpy()
    slots, first = [], 0
    for f, c, p in zip(fills, counts, pages):
        at = np.arange(f, f + c)
        slots.append(perm[first + at // bs] * bs + at % bs)
        first += p
    slots = torch.from_numpy(np.concatenate(slots)).cuda()
    n = slots.numel()
    key, value = torch.randn(2, n, kv_heads, dim, generator=g, device="cuda").to(dtype)
    cache = torch.randint(-127, 128, (2, nb, bs, kv_heads, dim), generator=g, device="cuda",
                          dtype=torch.int8)
    scales = (1 + 2 * torch.rand(2, nb, kv_heads, generator=g, device="cuda")) / 127
    positions = torch.randint(1024, (n,), generator=g, device="cuda")
    table = ops.rotary_table(1024, rot) if rot else None
    return key, value, cache, scales, slots, positions if rot else None, table


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("counts,fills,kv_heads,dim,bs,rot,interleaved", [
    ([1], [0], 8, 128, 16, 128, False),
    ([1] * 9, [0, 1, 7, 15, 16, 31, 3, 8, 2], 8, 128, 16, 128, False),
    ([1] * 600, [i % 16 for i in range(600)], 2, 64, 16, 32, True),   # the indexed path
    ([33, 1, 170, 16], [0, 15, 5, 0], 8, 128, 16, 128, False),
    ([900, 77, 1], [3, 0, 9], 4, 128, 16, 64, True),                  # indexed
    ([40, 5], [1, 60], 3, 256, 64, 256, False),
    ([40, 500], [1, 60], 3, 96, 64, 48, False),                       # indexed, 64 tokens a page
    ([11, 3], [0, 2], 1, 33, 5, 32, False),                           # scalar path
    ([11, 3], [0, 2], 1, 34, 5, 34, True),
    ([700], [0], 10, 30, 7, 0, False),
    ([20], [4], 40, 80, 32, 80, False),
])
def test_append_kv(cuda, dtype, counts, fills, kv_heads, dim, bs, rot, interleaved):
    key, value, cache, scales, slots, pos, table = append_problem(
        len(counts) + dim, counts, fills, kv_heads, dim, bs, DTYPES[dtype], rot)
    check_append(cuda, key, value, cache, scales, slots, bs, pos, table, interleaved)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("counts,fills,kv_heads,dim,bs,rot,interleaved", [
    ([700, 33], [0, 7], 5, 128, 32, 128, False),  # pages of more than 16 tokens
    ([600], [3], 6, 96, 32, 40, True),
    ([600, 70], [1, 0], 6, 64, 16, 24, False),    # rotary widths of 8 modulo 16
    ([560], [0], 12, 128, 16, 72, False),         # 24 heads for 8 warps
    ([14, 2], [2, 0], 9, 128, 16, 40, False),
    ([600], [0], 3, 128, 16, 12, True),           # half a piece rotated
    ([700, 33], [0, 7], 3, 256, 16, 256, False),  # a token for a whole warp
    ([600], [3], 2, 192, 16, 96, True),
    ([600], [0], 2, 256, 32, 64, False),
    ([700, 65], [5, 0], 3, 128, 64, 128, False),  # pages of 64 tokens
    ([640], [0], 2, 256, 64, 8, True),
])
def test_append_kv_whole_pages(cuda, dtype, counts, fills, kv_heads, dim, bs, rot, interleaved):
    key, value, cache, scales, slots, pos, table = append_problem(
        len(counts) + rot, counts, fills, kv_heads, dim, bs, DTYPES[dtype], rot)
    check_append(cuda, key, value, cache, scales, slots, bs, pos, table, interleaved)


@pytest.mark.parametrize("n", [50, 1400])
def test_append_kv_any_order_equal_slots_and_padding(cuda, n):
    """Tokens in shuffled order, slots that come twice, padding and slots
    outside the cache, on both paths; the rest of the cache stays."""
    key, value, cache, scales, slots, pos, table = append_problem(
        n, [n // 2, n - n // 2], [6, 0], 2, 128, 16, torch.bfloat16, 128)
    order = torch.randperm(n, generator=torch.Generator().manual_seed(n))
    slots = slots[order.cuda()]
    slots[::7] = slots[3]          # the same slot many times: the last one counts
    slots[5:9] = -1
    check_append(cuda, key, value, cache, scales, slots.clone(), 16, pos, table)
    slots[11] = cache.shape[1] * 16  # one past the end
    slots[12] = -2
    check_append(cuda, key, value, cache, scales, slots, 16, pos, table, error=3)


def test_append_kv_bad_position_skips_the_token(cuda):
    key, value, cache, scales, slots, pos, table = append_problem(
        5, [20], [0], 2, 128, 16, torch.float16, 128)
    pos[3], pos[18] = 1024, -1
    want_c, want_s = cache.clone(), scales.clone()
    from pagedkv_fusion import ops
    keep = [i for i in range(20) if i not in (3, 18)]
    ops.append_kv(key[keep], value[keep], want_c, want_s, slots[keep], 16, pos[keep], table)
    assert cuda.read_device_error() == 0
    ops.append_kv(key, value, cache, scales, slots, 16, pos, table)
    assert cuda.read_device_error() == 5
    assert torch.equal(cache, want_c) and torch.equal(scales, want_s)


def test_append_kv_special_values(cuda):
    """Zeros, huge and tiny values, infinities and NaN."""
    key, value, cache, scales, slots, _, _ = append_problem(
        6, [16, 16, 16, 16, 4, 4], [0, 0, 0, 0, 3, 3], 2, 128, 16, torch.float32, 0)
    key[:16] = 0
    key[16:32] *= 1e30
    key[32:48] *= 1e-41       # subnormal values and scale
    key[50, 0, 5] = float("nan")
    value[51, 1, 3] = float("-inf")
    key[65, 1, 7] = float("nan")   # in a started page: its scale stays
    key[70] = 0
    check_append(cuda, key, value, cache, scales, slots, 16)


def test_append_token_by_token_stays_readable(cuda):
    """A page filled by 40 single-token calls dequantizes within the rounding
    of its moves: each call that raises the scale re-rounds earlier codes, at
    most half a step of the scale at that time, and scales only grow."""
    from pagedkv_fusion import ops
    g = torch.Generator(device="cuda").manual_seed(9)
    n, bs = 40, 16
    key, value = torch.randn(2, n, 2, 64, generator=g, device="cuda")
    cache = torch.zeros(2, 4, bs, 2, 64, dtype=torch.int8, device="cuda")
    scales = torch.full((2, 4, 2), 50.0, device="cuda")  # left over: forgotten at offset 0
    table = ops.rotary_table(64, 64)
    pages = torch.tensor([2, 0, 3], device="cuda")
    grown = torch.zeros(2, 4, 2, device="cuda")
    for t in range(n):
        before = scales.clone()
        ops.append_kv(key[t:t + 1], value[t:t + 1], cache, scales, pages[t // bs:t // bs + 1] * bs + t % bs,
                      bs, torch.tensor([t], device="cuda"), table)
        grown += (scales > before) & torch.tensor(t % bs > 0, device="cuda")
    assert cuda.read_device_error() == 0
    assert int(grown.max()) >= 2
    got = (cache.double() * scales.double()[:, :, None, :, None])[:, pages].reshape(2, 48, 2, 64)[:, :n]
    want = torch.stack([rotate64(key.double(), table.double()[:n], False), value.double()])
    bound = (scales * (grown + 1) / 2)[:, pages].repeat_interleave(bs, 1)[:, :n, :, None]
    assert bool(((got - want).abs() <= bound * (1 + 1e-5)).all())


def test_append_kv_strided_views_stream_and_graph(cuda):
    """Views of a fused projection, on a side stream, and captured in a graph
    whose inputs change between replays."""
    from pagedkv_fusion import ops
    g = torch.Generator(device="cuda").manual_seed(10)
    n, kv, d, bs = 700, 4, 128, 16
    qkv = torch.randn(n, 8 * kv, d, generator=g, device="cuda").bfloat16()
    key, value = qkv[:, 4 * kv:5 * kv], qkv[:, 5 * kv:6 * kv]
    slots = torch.randperm(64 * bs, generator=g, device="cuda")[:n]
    pos = torch.arange(n, device="cuda")
    table = ops.rotary_table(n, d)
    cache = torch.randint(-127, 128, (2, 64, bs, kv, d), generator=g, device="cuda", dtype=torch.int8)
    scales = torch.rand(2, 64, kv, generator=g, device="cuda") / 50
    start_c, start_s = cache.clone(), scales.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        check_append(cuda, key, value, cache, scales, slots, bs, pos, table)
        graph = torch.cuda.CUDAGraph()
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        ops.append_kv(key, value, cache, scales, slots, bs, pos, table)
    for seed in (1, 2):
        qkv.copy_(torch.randn(n, 8 * kv, d, generator=g, device="cuda"))
        cache.copy_(start_c)
        scales.copy_(start_s)
        want_c, want_s = start_c.clone(), start_s.clone()
        ops.append_kv(key, value, want_c, want_s, slots, bs, pos, table)
        graph.replay()
        assert torch.equal(cache, want_c) and torch.equal(scales, want_s)
    assert cuda.read_device_error() == 0


def test_empty_calls(cuda):
    from pagedkv_fusion import ops
    table = ops.rotary_table(4, 64)
    none = torch.zeros(0, 4, 64, device="cuda")
    empty = torch.zeros(0, dtype=torch.int64, device="cuda")
    qo, ko = ops.qk_norm_rope(none, none, empty, table)
    assert qo.shape == ko.shape == (0, 4, 64)
    cache = torch.ones(2, 2, 16, 4, 64, dtype=torch.int8, device="cuda")
    ops.append_kv(none, none, cache, torch.ones(2, 2, 4, device="cuda"), empty, 16, empty, table)
    assert bool((cache == 1).all())


def test_host_inputs_are_staged(cuda):
    from pagedkv_fusion import ops
    r = np.random.default_rng(0)
    q = r.standard_normal((5, 2, 64)).astype(np.float32)
    table = ops.rotary_table(16, 64, device="cpu")
    qo, none = ops.qk_norm_rope(q, None, np.arange(5), table.numpy())
    assert isinstance(qo, np.ndarray) and none is None
    want = expected_qk(torch.from_numpy(q), torch.arange(5), table, None, 0, False)
    assert_rope_close(torch.from_numpy(qo), want, torch.float32)


def test_refusals(cuda):
    from pagedkv_fusion import ops
    q = torch.randn(4, 2, 64, device="cuda")
    pos = torch.arange(4, device="cuda")
    table = ops.rotary_table(8, 64)
    w = torch.ones(64, device="cuda")
    for call, msg in [
        (lambda: ops.qk_norm_rope(q.double(), None, pos, table), "float32"),
        (lambda: ops.qk_norm_rope(q, q.half(), pos, table), "q's type"),
        (lambda: ops.qk_norm_rope(q, q, pos[:3], table), "positions"),
        (lambda: ops.qk_norm_rope(q, q, pos.float(), table), "positions"),
        (lambda: ops.qk_norm_rope(q, q, pos, table.double()), "rotary"),
        (lambda: ops.qk_norm_rope(q, q, pos, torch.cat([table, table], 1)), "rotary"),
        (lambda: ops.qk_norm_rope(q, q, pos, table, w, None), "go together"),
        (lambda: ops.qk_norm_rope(q, q, pos, table, w, w.half()), "weights"),
        (lambda: ops.qk_norm_rope(q.clone().requires_grad_(), q, pos, table), "backward"),
    ]:
        with pytest.raises(RuntimeError, match=msg):
            call()
    cache = torch.zeros(2, 2, 16, 2, 64, dtype=torch.int8, device="cuda")
    scales = torch.ones(2, 2, 2, device="cuda")
    args = [q, q, cache, scales, pos, 16]
    for at, bad, msg in [(0, q[:, :1], "key/value"), (1, q.half(), "key/value"), (2, cache[0], "int8"),
                         (2, cache.transpose(1, 2), "contiguous"), (3, scales[:, :1], "contiguous"),
                         (4, pos[:2], "slot"), (4, pos.float(), "slot"), (5, 8, "block_size"),
                         (4, pos.cpu(), "CUDA")]:
        a = list(args)
        a[at] = bad
        with pytest.raises(RuntimeError, match=msg):
            ops.append_kv(*a)
    with pytest.raises(RuntimeError, match="go together"):
        ops.append_kv(*args, positions=pos)
    for kw in (dict(scaling="other"), dict(scaling="yarn"), dict(factor=0.0), dict(rotary_dim=63)):
        with pytest.raises(ValueError):
            ops.rotary_table(**{"max_positions": 4, "rotary_dim": 64, **kw})
