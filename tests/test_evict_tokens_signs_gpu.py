"""evict_tokens: scales of both signs and infinite ones, by the rule."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from test_evict_tokens_gpu import problem, run

pytestmark = pytest.mark.gpu


def by_the_rule(p, keep, sinks, recent):
    """The cache, scales and lengths after the eviction, from the kept places that it returned."""
    got, lens, kept = run(p, keep, sinks, recent)
    cache, scales = (p[k].cpu().numpy().copy() for k in ("kv_cache_int8", "scale_cache"))
    old_cache, old_scales = cache.copy(), scales.copy()
    bs = cache.shape[2]
    for i, n in enumerate(p["seq_lens"].tolist()):
        if n <= keep:
            continue
        pages, stay = p["block_tables"][i].cpu().numpy(), kept[i].cpu().numpy()
        for j in range(-(-keep // bs)):
            part = stay[j * bs:(j + 1) * bs]
            old = old_scales[:, pages[part // bs]]                   # [2, tokens, heads]
            codes = old_cache[:, pages[part // bs], part % bs].astype(np.float32)
            new = old.max(1, keepdims=True)
            with np.errstate(divide="ignore", invalid="ignore"):
                moved = np.rint(codes * (old / new)[..., None])
            moved = np.where((old < 0)[..., None], np.clip(moved, -127, 127), moved)
            codes = np.where((old < new)[..., None], moved, codes)
            cache[:, pages[j], :len(part)] = codes.astype(np.int8)
            scales[:, pages[j]] = new[:, 0]
    assert np.array_equal(got["scale_cache"].cpu().numpy(), scales)
    assert np.array_equal(got["kv_cache_int8"].cpu().numpy(), cache)
    return got, lens, kept


@pytest.mark.parametrize("dim", [64, 36, 33])
def test_scales_of_both_signs(cuda, dim):
    """A token whose scale is negative and smaller than its new page's has its codes clamped to
    -127 .. 127, -128 among the codes."""
    p = problem(21, [400, 90, 300], 2, dim, 16)
    p["kv_cache_int8"].random_(-128, 128)
    p["kv_cache_int8"][..., ::5] = -128
    sign = torch.where(torch.rand_like(p["scale_cache"]) < 0.4, -1.0, 1.0)
    p["scale_cache"] *= sign
    by_the_rule(p, 80, 3, 5)
    p["scale_cache"] = sign / 50  # old / new is -1 then
    by_the_rule(p, 80, 3, 5)
    p["scale_cache"] = -p["scale_cache"].abs()  # all negative: the one nearest to zero is the largest
    by_the_rule(p, 80, 3, 5)
