"""accumulate_attention held to the accuracy that it is built for with float32 queries (the limits:
test_chunk_accuracy_cpu.py), on each of its paths, the log denominators given and not.
"""

from __future__ import annotations

import pytest
import torch

from test_chunk_accuracy_cpu import SCORE_LIMIT
from test_chunk_accuracy_gpu import accuracy_problem, error, exact

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q_lens,keys,heads,kv_heads,dim,bs,order", [
    # the tensor-memory kernel; without denominators from the scores of a pass, or from the attention
    ([1] * 60, 8192, 40, 40, 64, 16, "mixed"), ([1] * 60, 8192, 32, 8, 128, 16, "falling"),
    ([1] * 4, 4096, 8, 8, 128, 32, "rising"), ([64], 16384, 32, 8, 128, 16, "mixed"),
    ([500, 4], 16384, 8, 2, 96, 16, "falling"),
    # pages and heads that only the warps' kernel takes
    ([1] * 60, 8192, 40, 40, 128, 24, "mixed"), ([64], 8192, 8, 2, 256, 16, "falling"),
])
def test_error_within_the_arithmetic(cuda, q_lens, keys, heads, kv_heads, dim, bs, order):
    from pagedkv_fusion import ops
    p = accuracy_problem(q_lens, keys, heads, kv_heads, dim, bs, order=order)
    want = exact(p)[2]
    lse = ops.chunk_attention(**p, return_lse=True)[1]
    args = {k: v for k, v in p.items() if not k.startswith("v_")}
    for given in (lse, None):
        weights = torch.zeros(p["k_cache_q"].shape[:2], device="cuda")
        ops.accumulate_attention(weights, **args, lse=given)
        got = weights[p["block_tables"][0].long()].flatten()[:keys]
        off = error(got, want)
        assert off <= SCORE_LIMIT[max(dim, 128)], (given is None, off)
    assert cuda.read_device_error() == 0
