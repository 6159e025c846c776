"""prefill_attention's cu_seqlens: lists of more than 32 sequences that do not
ascend within the tensors are reported wherever the mistake is.  Entries are cut
to the tensors, those of the rows also to the largest before them: every row is
written, by one sequence.  Rows in front of the first
sequence are zero, as those behind the last are.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from test_prefill_gpu import cumulative, problem

pytestmark = pytest.mark.gpu

LENS = [3] * 70


def entries(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("at,value", [
    (1, 200), (31, -1), (32, 5), (33, 500), (40, 3), (69, 211), (69, 0), (70, 1000), (70, 0),
])
def test_a_bad_entry_is_reported_wherever_it_is(cuda, at, value):
    from pagedkv_fusion import ops
    q, k, v = problem(at, LENS, LENS, 4, 2, 64, "bf16")
    good = cumulative(LENS)
    bad = good.clone()
    bad[at] = value
    ops.prefill_attention(q, k, v, good, 0.1)
    assert cuda.read_device_error() == 0
    for cu, ck in ((bad, None), (good, bad), (bad, good)):
        ops.prefill_attention(q, k, v, cu, 0.1, cu_seqlens_k=ck)
        assert cuda.read_device_error() == 6
        ops.prefill_attention(q, k, v, good, 0.1)  # and it does not stay
        assert cuda.read_device_error() == 0


def test_empty_sequences_and_thousands_are_no_mistake(cuda):
    from pagedkv_fusion import ops
    for lens in ([0] * 40 + [5] + [0] * 40 + [7], [1, 0, 2] * 700):
        q, k, v = problem(len(lens), lens, lens, 4, 2, 64, "f16")
        ops.prefill_attention(q, k, v, cumulative(lens), 0.1)
        assert cuda.read_device_error() == 0
    ops.prefill_attention(q, k, v, cumulative([]), 0.1)
    assert cuda.read_device_error() == 0
    ops.prefill_attention(q, k, v, entries([-1]), 0.1)
    assert cuda.read_device_error() == 6


def ragged(rng, n, top):
    """A list of n + 1 entries that rises, falls and leaves [0, top]."""
    up = np.sort(rng.integers(0, top + 1, n + 1))
    for at in rng.integers(0, n + 1, max(2, n // 8)):
        up[at] = rng.integers(-20, top + 100)
    return up.tolist()


def cut(q_list, k_list, top):
    """The same sequences as good lists: the keys of each laid out anew, as the
    places of its rows in the key tensor."""
    q_cut = np.maximum.accumulate(np.clip(q_list, 0, top)).tolist()
    ends = np.clip(k_list, 0, top).tolist()
    keys = [np.arange(a, max(a, b)) for a, b in zip(ends, ends[1:])]
    return q_cut, [0] + np.cumsum([len(x) for x in keys]).tolist(), np.concatenate(keys).astype(int)


def filled_with_nan(t):
    """Freed memory of t's size that holds NaN, which the next output gets."""
    t = torch.full_like(t, float("nan"))
    torch.cuda.synchronize()
    del t


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("q_list,k_list", [
    ([0, 300] * 20 + [300], None),     # the same rows again and again: more items than the grid
    ([0, 300, 0, 0, 150, 100, 300], None),
    ([0, 100, 50, 400], [0, 100, 200, 350]),
    ([0, 100, 200, 350], [0, 200, 100, 400]),
    ([0, 900, 120], None),
    ([0, 100, -2 ** 31, 2 ** 31 - 1, 400], None),
    ([0, 100, 400], [5, -2 ** 31, 2 ** 31 - 1]),
    ("ragged", "ragged"),
    ("ragged", None),
])
def test_falling_entries_share_no_rows(cuda, dtype, q_list, k_list):
    from pagedkv_fusion import ops
    rng = np.random.default_rng(3)
    q, k, v = problem(7, [400], [400], 8, 2, 64, dtype)
    for n in ((5, 40, 130) if q_list == "ragged" else (0,)):
        cq = ragged(rng, n, 400) if n else q_list
        ck = ragged(rng, n, 400) if k_list == "ragged" else (k_list or cq)
        q_cut, k_cut, at = cut(cq, ck, 400)
        want, lse = ops.prefill_attention(q, k[at], v[at], entries(q_cut), 0.1,
                                          cu_seqlens_k=entries(k_cut), return_lse=True)
        assert cuda.read_device_error() == 0
        filled_with_nan(q)
        out, got = ops.prefill_attention(q, k, v, entries(cq), 0.1, cu_seqlens_k=entries(ck),
                                         return_lse=True)
        assert cuda.read_device_error() == 6
        first = q_cut[0]  # (rows in front of the first sequence are not its)
        assert torch.equal(out[first:], want[first:]) and torch.equal(got[first:], lse[first:])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows,cu", [
    (100, [10, 60]), (100, [10, 60, 100]), (100, [100]), (100, [37]), (100, [100, 100, 100]),
    (5000, [4990, 4995]), (700, [1] + [1 + 22 * i for i in range(1, 31)]),
    (700, [300] + [300 + 10 * i for i in range(1, 41)]), (300, [500, 600]),
])
def test_rows_in_front_of_the_first_sequence(cuda, dtype, rows, cu):
    import math
    from pagedkv_fusion import ops
    q, k, v = problem(rows, [rows], [rows], 8, 2, 64, dtype)
    filled_with_nan(q)
    out, lse = ops.prefill_attention(q, k, v, entries(cu), 0.1, return_lse=True)
    a, b = min(cu[0], rows), min(cu[-1], rows)
    assert cuda.read_device_error() == (6 if cu[-1] > rows else 0)
    for rest in (slice(0, a), slice(b, None)):
        assert bool((out[rest] == 0).all()) and bool((lse[rest] == -math.inf).all())
    if b > a:
        want, wlse = ops.prefill_attention(q[a:b], k[a:b], v[a:b], entries(cu) - a, 0.1, return_lse=True)
        assert torch.equal(out[a:b], want) and torch.equal(lse[a:b], wlse)
