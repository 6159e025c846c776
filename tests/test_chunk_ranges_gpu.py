"""chunk_attention where maxima, units of V and signs move, held to the tolerance of
test_chunk_gpu.py.
"""

from __future__ import annotations

import pytest
import torch

from test_chunk_gpu import check, problem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("q_lens,lens,heads,kv_heads,dim,each", [
    ([200], [900], 8, 1, 128, 1), ([200], [900], 8, 1, 64, 1),  # both row tiles, every tile a new unit
    ([16], [5000], 8, 1, 128, 4),                              # even and odd tiles apart
    ([300], [2100], 4, 2, 96, 2), ([3], [900], 8, 2, 128, 1),   # two heads; few rows
])
def test_rising_v_scales_beside_rising_scores(cuda, dtype, q_lens, lens, heads, kv_heads, dim, each):
    """Later tiles of 128 keys have larger V scales and, for every other row alone, scores far
    above the earlier ones: what was gathered so far is moved twice within a tile, by the new unit
    of V and, beside rows whose maximum moves, by nothing."""
    p = problem(31, q_lens, lens, heads, kv_heads, dim, 16, dtype, spread=0.1)
    p["q"][:, ::2] *= 2.0 ** -12  # these attend evenly
    pages = p["block_tables"][0].long()
    step = (torch.arange(len(pages), device="cuda") // (8 * each)).float()[:, None]
    p["k_scale"][pages] *= 0.1 * 2.0 ** step
    p["v_scale"][pages] *= 1.7 ** step
    check(p)
    p["v_scale"][pages] *= 1.7 ** -step * 2.0 ** -(step % 3)  # and falling again
    check(p)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("q_lens,lens,heads,kv_heads,dim,bs", [
    ([1, 2], [900, 333], 8, 2, 128, 16), ([200], [1500], 8, 2, 128, 16), ([90, 1], [1500, 40], 8, 2, 64, 32),
    ([16], [5000], 8, 1, 128, 16), ([1, 40], [300, 90], 8, 2, 160, 5),
])
def test_scale_of_any_sign(cuda, dtype, q_lens, lens, heads, kv_heads, dim, bs):
    """A negative sm_scale turns the scores' order around, for all keys or (with negative K scales)
    for some; the scores spread over tens of powers of two.  With 0 all keys weigh the same."""
    for spread, factor in ((0.1, -1.0), (0.5, -1.0), (0.5, -4.0), (0.5, 0.0)):
        p = problem(32, q_lens, lens, heads, kv_heads, dim, bs, dtype, spread=spread)
        p["sm_scale"] *= factor
        check(p)
        p["k_scale"][::3] *= -1
        check(p)


def test_values_that_are_not_finite_reach_rows_that_see_them(cuda):
    """However little weight they have there, and in whichever part of the keys they are."""
    from pagedkv_fusion import ops
    for q_lens, lens, heads, kv_heads in (([1], [60], 8, 2), ([1], [300], 8, 2), ([1, 2], [900, 200], 8, 2),
                                          ([1], [9000], 8, 2), ([300], [900], 8, 2), ([16], [6000], 8, 1)):
        p = problem(33, q_lens, lens, heads, kv_heads, 128, 16, "f32", spread=0.0)
        p["q"].abs_().add_(0.5).mul_(4)  # 200 nats from page to page
        p["k_cache_q"].fill_(-100)
        p["k_cache_q"][p["block_tables"][0, 0].long()] = 100  # the first page has all of the weight
        want = ops.chunk_attention(**p)
        assert bool(torch.isfinite(want).all())
        for page in sorted({1, lens[0] // 32, (lens[0] - q_lens[0]) // 16 - 1} - {0}):
            for bad in (float("inf"), float("nan")):
                broken = dict(p, v_scale=p["v_scale"].clone())
                broken["v_scale"][p["block_tables"][0, page].long()] = bad
                out = ops.chunk_attention(**broken)
                assert not bool(torch.isfinite(out[:q_lens[0]]).any()), (lens, page, bad)
                assert torch.equal(out[q_lens[0]:], want[q_lens[0]:])


def test_cache_without_pages(cuda):
    """Nothing is cached: every row is zero; lengths and table entries all the same are errors."""
    from pagedkv_fusion import ops
    for q_lens, lens, kv_heads, bs in (([1, 2], [0, 0], 2, 16), ([300, 40], [0, 0], 2, 16), ([300], [600], 1, 16),
                                       ([2], [40], 2, 16), ([40], [60], 2, 5)):
        p = problem(34, q_lens, lens, 8, kv_heads, 128, bs, "bf16", wide=1)
        for name in ("k_cache_q", "v_cache_q", "k_scale", "v_scale"):
            p[name] = p[name][:0].clone()
        out, lse = ops.chunk_attention(**p, return_lse=True)
        assert bool((out == 0).all()) and bool((lse == -float("inf")).all())
        assert cuda.read_device_error() == (1 if max(lens) else 0)
        args = {k: v for k, v in p.items() if not k.startswith("v_")}
        weights = torch.zeros(0, bs, device="cuda")
        for given in (lse, None):
            ops.accumulate_attention(weights, **args, lse=given)
        assert cuda.read_device_error() in ((0, 1) if max(lens) else (0,))
