"""accumulate_attention against the softmax probabilities of 64 bits, summed per cached token.

Tolerance: a probability's relative error is its score's (t, see test_chunk_gpu.py) and its
denominator's (t again and n 2^-23, or 2^-22 |lse| where it was given), with 2^-18 for the
exponentials and logarithms; a power of two common to 256 rows leaves a score 2^-35 of the
largest query times the keys; sums over the rows are fp32 (2^-22), meet in steps of 2^-38 (half
of one for each of the parts, taken as 2^-30), and are added to what was there (2^-23).
"""

from __future__ import annotations

import math

import pytest
import torch

from test_chunk_gpu import problem, reference

pytestmark = pytest.mark.gpu


def call(p, weights, lse=None):
    from pagedkv_fusion import ops
    args = {k: v for k, v in p.items() if not k.startswith("v_")}
    assert ops.accumulate_attention(weights, **args, lse=lse) is None
    return weights


def expected(p, start):
    want, tol = start.double().clone(), 2.0 ** -30 + torch.zeros_like(start).double()
    bs = start.shape[1]
    _, _, lse, _, parts = reference(p)
    H = p["q"].shape[1]
    k_most = 127 * p["k_scale"].double().abs().max()
    loose = 2.0 ** -35 * p["q"].double().abs().max() * k_most * p["q"].shape[2] * abs(p["sm_scale"])
    at = torch.arange(p["block_tables"].shape[1] * bs, device="cuda")
    for i, j, rows, n, w, t in parts:
        slots = p["block_tables"][i].long()[at[:n] // bs] * bs + at[:n] % bs
        rel = 2 * t + n * 2.0 ** -23 + 2.0 ** -18 + loose + 2.0 ** -22 * lse[rows, j].abs().nan_to_num(0, 0, 0)
        want.view(-1).index_add_(0, slots, w.sum(0) / H)
        tol.view(-1).index_add_(0, slots, (w * (rel[:, None] + 2.0 ** -22)).sum(0) / H)
    return want, tol + 2.0 ** -23 * want.abs()


def check(p, given=False, error=0):
    from pagedkv_fusion import _C, ops
    g = torch.Generator(device="cuda").manual_seed(1)
    start = torch.rand(p["k_cache_q"].shape[:2], generator=g, device="cuda")
    lse = ops.chunk_attention(**p, return_lse=True)[1] if given else None
    got = call(p, start.clone(), lse)
    assert _C.read_device_error() == error
    want, tol = expected(p, start)
    bad = ~((got.double() - want).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float((got - want).abs().max()), bad.nonzero()[:5].tolist())
    assert torch.equal(call(p, start.clone(), lse), got)  # the same bits every time
    return got


SHAPES = [
    ([1], [1], 1, 1, 32, 16), ([1] * 7, [0, 1, 15, 16, 17, 300, 64], 32, 8, 128, 16),
    ([1] * 20, [3 + 67 * i for i in range(20)], 16, 2, 96, 8), ([1] * 3, [900, 40, 260], 8, 8, 64, 32),
    ([3, 0, 8, 2], [50, 9, 1000, 2], 12, 4, 128, 32), ([300], [300], 8, 2, 128, 16),
    ([70, 1, 33], [900, 600, 33], 32, 8, 128, 16), ([40], [3000], 40, 40, 64, 64), ([50], [20], 8, 2, 128, 16),
    ([9], [77], 33, 1, 128, 16), ([60], [300], 4, 2, 160, 16), ([1, 40], [500, 60], 8, 1, 256, 16),
    ([33, 1, 1], [200, 9, 70], 8, 2, 128, 1), ([100], [333], 8, 4, 128, 24), ([1] * 4, [50, 7, 0, 200], 8, 2, 64, 5),
    ([600, 2], [700, 1400], 8, 2, 64, 5),
]


@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("q_lens,lens,heads,kv_heads,dim,bs", SHAPES)
def test_matches_reference(cuda, dtype, q_lens, lens, heads, kv_heads, dim, bs, given):
    check(problem(1, q_lens, lens, heads, kv_heads, dim, bs, dtype, wide=len(lens) % 3), given)


def test_every_token_spreads_a_weight_of_one(cuda):
    for q_lens, lens in (([1] * 30, [20 + 50 * i for i in range(30)]), ([700, 5], [900, 2000])):
        p = problem(2, q_lens, lens, 16, 4, 128, 16)
        total = float(call(p, torch.zeros(p["k_cache_q"].shape[:2], device="cuda")).double().sum())
        assert abs(total / sum(q_lens) - 1) < 1e-5


@pytest.mark.parametrize("q_lens,lens,bs", [([1] * 6, [100] * 6, 16), ([50, 1, 70], [100] * 3, 16),
                                            ([300, 1, 90], [700] * 3, 16),
                                            ([1, 3], [40, 40], 5)])
def test_shared_pages_gather_from_all(cuda, q_lens, lens, bs):
    p = problem(3, q_lens, lens, 8, 2, 128, bs)
    p["block_tables"][1:] = p["block_tables"][0]  # all of them
    p["block_tables"][-1, 0] = p["block_tables"][0, 1]  # and one page twice in a table
    for given in (False, True):
        check(p, given)


def test_rows_of_other_magnitudes(cuda):
    for q_lens in ([1, 1], [60, 3]):
        p = problem(4, q_lens, [500, 80], 8, 2, 128, 16, "f32")
        p["q"] *= torch.tensor([2.0 ** -30, 1.0, 8.0, 0.0, 2.0 ** -5, 3.0, 2.0 ** -12, 1.0],
                               device="cuda").view(1, -1, 1)
        p["k_scale"][::3] *= -1
        p["k_scale"][::7] = 0.0
        for given in (False, True):
            check(p, given)


def test_not_finite(cuda):
    """NaN of a row or a scale reaches the weights of the tokens that it concerns, others stay."""
    for q_lens, lens in (([1, 1], [100, 60]), ([50, 3], [100, 60]), ([400, 3], [900, 60])):
        p = problem(5, q_lens, lens, 8, 2, 128, 16, "f16")
        zero = torch.zeros(p["k_cache_q"].shape[:2], device="cuda")
        want = call(p, zero.clone())
        pages = [p["block_tables"][i, :-(-n // 16)].long() for i, n in enumerate(lens)]
        broken = dict(p, q=p["q"].clone())
        broken["q"][-1, 0, 3] = math.nan  # the last sequence's last token
        got = call(broken, zero.clone())
        assert torch.equal(got[pages[0]], want[pages[0]])
        assert bool(got[pages[1]].view(-1)[:lens[1]].isnan().all())
        # a scale on the page of the last tokens: rows in front of them add what they did
        broken = dict(p, k_scale=p["k_scale"].clone())
        broken["k_scale"][pages[0][-1]] = math.nan
        got = call(broken, zero.clone())
        assert torch.equal(got[pages[1]], want[pages[1]])
        assert bool(got[pages[0]].view(-1)[:lens[0]].isnan().all())
        # a row without lse adds nothing, rows behind all sequences are not read
        from pagedkv_fusion import ops
        lse = ops.chunk_attention(**p, return_lse=True)[1]
        lse[:q_lens[0]] = -math.inf
        assert bool((call(p, zero.clone(), lse)[pages[0]] == 0).all())


def test_bad_pages_lengths_and_nothing(cuda):
    for q_lens, lens, bs in (([1, 2], [100, 60], 16), ([60, 2], [100, 60], 16), ([300, 40], [700, 2000], 16),
                             ([1, 2], [100, 60], 5)):
        p = problem(6, q_lens, lens, 8, 2, 128, bs, "f32")
        zero = torch.zeros(p["k_cache_q"].shape[:2], device="cuda")
        want = call(p, zero.clone())
        pages = [p["block_tables"][i, :-(-n // bs)].long() for i, n in enumerate(lens)]
        for bad in (-1, zero.shape[0], 2 ** 31 - 1):
            broken = dict(p, block_tables=p["block_tables"].clone())
            broken["block_tables"][0, 1] = bad
            got = call(broken, zero.clone())
            assert cuda.read_device_error() == 1
            assert torch.equal(got[pages[1]], want[pages[1]])
            assert bool((got[pages[0][1]] == 0).all())
            total = float(got[pages[0]].double().sum())
            assert abs(total / q_lens[0] - 1) < 1e-5  # the others take its share
        long = dict(p, seq_lens=p["seq_lens"].clone(), block_tables=p["block_tables"].clamp(min=0))
        long["seq_lens"][0] = 2 ** 31 - 1
        call(long, zero.clone())
        assert cuda.read_device_error() == 4
        for none in (dict(seq_lens=p["seq_lens"] * 0), dict(cu_seqlens=p["cu_seqlens"] * 0),
                     dict(seq_lens=p["seq_lens"] * 0 - 3)):
            assert bool((call(dict(p, **none), zero.clone()) == 0).all())
        empty = dict(p, q=p["q"][:0], cu_seqlens=p["cu_seqlens"] * 0)
        assert bool((call(empty, zero.clone()) == 0).all())
        assert bool((call(dict(p, block_tables=p["block_tables"][:, :0], seq_lens=p["seq_lens"] * 0),
                          zero.clone()) == 0).all())
    assert cuda.read_device_error() == 0


def test_graph_and_streams(cuda):
    from pagedkv_fusion import ops
    problems = [problem(7, [1] * 5, [300, 40, 1, 64, 900], 8, 2, 128, 16, "bf16"),
                problem(8, [64], [1500], 32, 8, 128, 16, "f16"),
                problem(10, [300, 2], [700, 40], 8, 2, 128, 16, "f32")]
    start = [torch.rand(p["k_cache_q"].shape[:2], device="cuda") for p in problems]
    lses = [None, ops.chunk_attention(**problems[1], return_lse=True)[1], None]
    want, graphs, buffers = [], [], []
    for p, s, lse in zip(problems, start, lses):
        want.append(call(p, s.clone(), lse))
        w = s.clone()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(p, w, lse)
        graphs.append(g)
        buffers.append(w)
    streams = [torch.cuda.Stream() for _ in problems]
    for _ in range(3):
        for w, s in zip(buffers, start):
            w.copy_(s)
        torch.cuda.synchronize()
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        eager = [call(p, s.clone(), lse) for p, s, lse in zip(problems, start, lses)]
        torch.cuda.synchronize()
        for w, e, x in zip(buffers, eager, want):
            assert torch.equal(w, x) and torch.equal(e, x)


def test_refusals(cuda):
    from pagedkv_fusion import ops
    p = problem(9, [2, 1], [30, 9], 4, 2, 64, 16, "f16")
    args = {k: v for k, v in p.items() if not k.startswith("v_")}
    w = torch.zeros(p["k_cache_q"].shape[:2], device="cuda")
    lse = torch.zeros(3, 4, device="cuda")
    for weights, change, message in [
            (w.double(), {}, "weights"), (w[:-1], {}, "weights"), (w.T.contiguous().T, {}, "contiguous"),
            (w, dict(lse=lse[:2]), "lse"), (w, dict(lse=lse.double()), "lse"),
            (w, dict(q=p["q"].double()), "q must be"), (w, dict(k_cache_q=p["k_cache_q"].float()), "int8"),
            (w, dict(cu_seqlens=p["cu_seqlens"][1:]), "cu_seqlens"), (w.cpu(), {}, "CUDA"),
            (w.clone().requires_grad_(), {}, "no backward")]:
        with pytest.raises(RuntimeError, match=message):
            ops.accumulate_attention(weights, **dict(args, **change))
    ops.accumulate_attention(w, **args, lse=lse.T.contiguous().T)
    assert cuda.read_device_error() == 0
