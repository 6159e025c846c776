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


def keys_without_weight(p, seq, head):
    """The slots to which the last token of `seq` gives a weight of 0 in 64 bits with `head`."""
    bs, n = p["k_cache_q"].shape[1], int(p["seq_lens"][seq])
    pages, at = p["block_tables"][seq].long(), torch.arange(n, device="cuda")
    group = p["q"].shape[1] // p["k_scale"].shape[1]
    h, t = head // group, pages[:-(-n // bs)]
    k = (p["k_cache_q"][t, :, h].double() * p["k_scale"][t, h].double()[:, None, None]).flatten(0, 1)[:n]
    weight = torch.softmax(k @ p["q"][int(p["cu_seqlens"][seq + 1]) - 1, head].double() * p["sm_scale"], 0)
    calm = torch.ones(p["k_cache_q"].shape[:2], dtype=torch.bool, device="cuda")
    calm[pages[at // bs], at % bs] = weight == 0
    return calm


SHAPES = [([1, 1], [700, 300], 16), ([60, 3], [700, 300], 16), ([300, 5], [900, 300], 32), ([60, 3], [700, 300], 5)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("q_lens,lens,bs", SHAPES)
def test_a_huge_row_leaves_the_others_their_weights(cuda, dtype, q_lens, lens, bs):
    """One head of one token is 2^66 (fp16: 2^10) times as large as the others, which add what they
    add beside a row of their own size: operands keep 2^-26 of a row's largest, of scores whose
    terms' magnitudes sum to 300, 4.5e-6, so 2^-15 of a weight.  (The row's own keys, one
    of which has all of its weight, are left out: its scores' last place is more than 1.)"""
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
        assert bool(((rows_alone(big, others, all_lse) - want).abs() <= 2.0 ** -15 * want).all()), factor
        calm = keys_without_weight(big, len(q_lens) - 1, 5)
        assert int((calm & (want > 0)).sum()) > 0.9 * int((want > 0).sum())
        for given in (all_lse, None):
            got = call(big, torch.zeros_like(want), given)
            assert bool(((got - want).abs() <= 2.0 ** -15 * want)[calm].all()), (factor, given is None)


def test_magnitudes_of_all_sizes(cuda):
    """Every row of a unit has a magnitude of its own, zero and 2^-60 to 2^12 among them."""
    for q_lens, lens, heads in (([64], [300], 8), ([1, 1], [500, 80], 8), ([300], [700], 4)):
        p = problem(42, q_lens, lens, heads, 2, 128, 16, "f32")
        rows = p["q"].shape[0] * heads
        power = torch.randint(-60, 4, (rows,), generator=torch.Generator().manual_seed(1))
        p["q"] *= torch.where(power % 7 == 0, 0.0, 2.0 ** power.double()).float().view(-1, heads, 1).cuda()
        for given in (False, True):
            check(p, given)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("q_lens,lens,bs", SHAPES)
def test_negative_scale(cuda, dtype, q_lens, lens, bs):
    p = problem(44, q_lens, lens, 8, 2, 128, bs, dtype)
    p["sm_scale"] *= -3
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
