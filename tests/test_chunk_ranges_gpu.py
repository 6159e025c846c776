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
