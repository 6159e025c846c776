"""accumulate_attention: rows of very different magnitudes, rows that add nothing, the largest sums."""

from __future__ import annotations

import math

import pytest
import torch

from test_chunk_gpu import problem
from test_weights_gpu import call, check

pytestmark = pytest.mark.gpu


def rows_alone(p, rows, lse):
    """The weights from the tokens and heads `rows` (a mask) alone: the others' lse is -inf."""
    only = torch.where(rows, lse, -math.inf)
    return call(p, torch.zeros(p["k_cache_q"].shape[:2], device="cuda"), only)


SHAPES = [([1, 1], [700, 300], 16), ([60, 3], [700, 300], 16), ([300, 5], [900, 300], 32), ([60, 3], [700, 300], 5)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("q_lens,lens,bs", SHAPES)
def test_a_huge_row_leaves_the_others_their_weights(cuda, dtype, q_lens, lens, bs):
    """One head of one token is 2^66 (fp16: 2^10) times as large as the others: what they add is
    what they add beside a row of their own size, within fp32's sums (the most any 256 rows' order
    could change, 2^-15 of a weight)."""
    from pagedkv_fusion import ops
    p = problem(41, q_lens, lens, 8, 2, 128, bs, dtype)
    lse = ops.chunk_attention(**p, return_lse=True)[1]
    others = torch.ones_like(lse, dtype=torch.bool)
    others[-1, 5] = False
    want = rows_alone(p, others, lse)
    for factor in ([2.0 ** 66, 2.0 ** 20] if dtype != "f16" else [2.0 ** 10]):
        big = dict(p, q=p["q"].clone())
        big["q"][-1, 5] *= factor
        all_lse = ops.chunk_attention(**big, return_lse=True)[1]
        assert torch.equal(all_lse[others], lse[others])
        for given in (all_lse, None):
            got = call(big, torch.zeros_like(want), given)
            one = rows_alone(big, ~others, all_lse)
            assert bool(torch.isfinite(got).all())
            assert bool(((got - one - want).abs() <= 2.0 ** -15 * (want + one)).all()), (factor, given is None)


def test_magnitudes_of_all_sizes(cuda):
    """Every row of a unit has a magnitude of its own, zero and 2^-60 to 2^12 among them."""
    for q_lens, lens, heads in (([64], [300], 8), ([1, 1], [500, 80], 8), ([300], [700], 4)):
        p = problem(42, q_lens, lens, heads, 2, 128, 16, "f32")
        rows = p["q"].shape[0] * heads
        power = torch.randint(-60, 4, (rows,), generator=torch.Generator().manual_seed(1))
        p["q"] *= torch.where(power % 7 == 0, 0.0, 2.0 ** power.double()).float().view(-1, heads, 1).cuda()
        for given in (False, True):
            check(p, given)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("q_lens,lens,bs", SHAPES)
def test_rows_without_denominator_add_nothing(cuda, dtype, q_lens, lens, bs):
    """Whatever their queries hold."""
    from pagedkv_fusion import ops
    p = problem(43, q_lens, lens, 8, 2, 128, bs, dtype)
    lse = ops.chunk_attention(**p, return_lse=True)[1]
    some = torch.rand(lse.shape, device="cuda") < 0.7
    want = rows_alone(p, some, lse)
    for bad in (math.nan, math.inf):
        broken = dict(p, q=torch.where(some[..., None], p["q"], bad))
        assert torch.equal(rows_alone(broken, some, lse), want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("q_lens,lens,bs", SHAPES)
def test_negative_scale(cuda, dtype, q_lens, lens, bs):
    p = problem(44, q_lens, lens, 8, 2, 128, bs, dtype)
    p["sm_scale"] *= -3
    for given in (False, True):
        check(p, given)


@pytest.mark.parametrize("bs", [16, 5])
def test_the_largest_sum(cuda, bs):
    """2^25 rows, the most of a call, with all their weight on one token: 2^22 sequences of 8 heads
    that share a page and have one token each."""
    S, H, D = 1 << 22, 8, 32
    q = torch.zeros(S, H, D, dtype=torch.float16, device="cuda")
    k = torch.zeros(2, bs, 1, D, dtype=torch.int8, device="cuda")
    args = dict(q=q, k_cache_q=k, k_scale=torch.ones(2, 1, device="cuda"),
                block_tables=torch.ones(S, 1, dtype=torch.int32, device="cuda"),
                seq_lens=torch.ones(S, dtype=torch.int32, device="cuda"),
                cu_seqlens=torch.arange(S + 1, dtype=torch.int32, device="cuda"), sm_scale=1.0)
    got = call(args, torch.zeros(2, bs, device="cuda"), torch.zeros(S, H, device="cuda"))
    assert float(got[1, 0]) == S and float(got.sum()) == S
    assert cuda.read_device_error() == 0
