"""prefill_attention's cu_seqlens: lists of more than 32 sequences that do not
ascend within the tensors are reported wherever the mistake is.
"""

from __future__ import annotations

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
