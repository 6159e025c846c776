"""evict_tokens: scales of both signs and infinite ones, by the rule; long sequences whose sort
keys are read from the weights again and again."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from test_evict_tokens_gpu import check, problem, run

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


def test_infinite_scales(cuda):
    """A page with a token of infinite scale takes it: codes of finite scales become 0, the others
    stay."""
    p = problem(22, [200, 150], 2, 64, 16)
    p["scale_cache"][0, ::3] = float("inf")
    p["scale_cache"][1, 1::4] = float("inf")
    got, _, kept = by_the_rule(p, 60, 2, 2)
    page = got["kv_cache_int8"][0, p["block_tables"][0, 0].long()]
    old = p["scale_cache"][0, p["block_tables"][0, kept[0, :16].long() // 16].long(), 0]
    if bool(old.isinf().any()):
        assert bool((page[~old.isinf(), 0] == 0).all()) and bool((page[old.isinf(), 0] != 0).any())


@pytest.mark.parametrize("long,others,keep", [(50000, 75, 20000), (98304, 74, 98303), (49153, 148, 3)])
def test_keys_that_do_not_fit_on_chip(cuda, long, others, keep):
    """One long sequence beside so many that each has one CTA."""
    p = problem(23, [long] + [40] * others, 1, 32, 16)
    check(p, keep, min(keep, 2) - 1, 1)
    p["weights"].copy_(torch.round(p["weights"] * 4) / 4)  # few values: the earlier token stays
    check(p, keep, 0, 0)
