"""shared_prefix_attention held to the accuracy that it is built for: the root
mean square of its error within the limits of the arithmetic (derived, and
shown to tell a loss of precision, in test_prefix_accuracy_cpu.py).  V codes
have one sign.
"""

from __future__ import annotations

import pytest
import torch

from test_prefix_accuracy_cpu import FAR, LIMIT, NEAR, SPREAD
from test_prefix_gpu import problem

pytestmark = pytest.mark.gpu


def accuracy_problem(prefix, seqs, heads, kv_heads, dim, bs, order):
    """Scores of standard deviation SPREAD, the pages' K scales uneven, or
    rising or falling along the prefix; two own tokens a sequence."""
    p = problem(prefix + seqs, prefix, [2] * seqs, heads, kv_heads, dim, bs)
    for name in ("k_scale", "v_scale"):
        p[name].uniform_(0.5, 1.5)
    if order != "mixed":
        ramp = torch.linspace(0.1, 1.5, len(p["prefix_table"]), device="cuda")[:, None]
        p["k_scale"][p["prefix_table"].long()] = ramp if order == "rising" else ramp.flip(0)
    p["k_scale"] *= SPREAD / 73.3
    p["v_scale"] /= 64
    p["v_cache_q"].random_(1, 128)
    return p


def exact(p):
    q = p["q"].double()
    kv, bs = p["k_cache_q"].shape[2], p["k_cache_q"].shape[1]
    group, n0 = q.shape[1] // kv, int(p["prefix_len"])
    out = torch.zeros_like(q)

    def tokens(cache, scale, pages, h):  # [..., pages] -> [..., tokens, D]
        t = pages.long()
        return (cache[t, :, h].double() * scale[t, h].double()[..., None, None]).flatten(-3, -2)

    for h in range(kv):
        k0, v0 = (tokens(p[c], p[s], p["prefix_table"], h)[:n0]
                  for c, s in (("k_cache_q", "k_scale"), ("v_cache_q", "v_scale")))
        k1, v1 = (tokens(p[c], p[s], p["block_tables"], h)[:, :2]
                  for c, s in (("k_cache_q", "k_scale"), ("v_cache_q", "v_scale")))
        rows = q[:, h * group:(h + 1) * group]
        w = torch.softmax(torch.cat([rows @ k0.T, rows @ k1.transpose(1, 2)], 2) * p["sm_scale"], 2)
        out[:, h * group:(h + 1) * group] = w[..., :n0] @ v0 + w[..., n0:] @ v1
    return out


@pytest.mark.parametrize("flush,prefix,seqs,heads,kv_heads,dim,bs,order", [
    # O's sum in tensor memory (one row tile, or head_dim up to 64)
    (NEAR, 4096, 8, 8, 8, 128, 16, "mixed"),        # parts of 2 tiles
    (NEAR, 16384, 20, 40, 40, 128, 16, "mixed"),    # of 19
    (NEAR, 16384, 20, 40, 40, 128, 16, "rising"),
    (NEAR, 32768, 130, 40, 40, 64, 32, "mixed"),    # of 37; two row tiles
    (NEAR, 16384, 20, 40, 40, 96, 16, "falling"),
    # in global memory (two row tiles of head_dim above 64): taken in every 5 tiles
    (FAR, 32768, 64, 32, 8, 128, 16, "mixed"),      # parts of 14 or 15 tiles: twice
    (FAR, 16384, 130, 40, 40, 128, 24, "mixed"),    # of 19: three times
    (FAR, 32768, 130, 40, 40, 128, 16, "mixed"),    # of 37: seven times
    (FAR, 32768, 130, 40, 40, 128, 16, "rising"),   # maxima move after each
    (FAR, 32768, 130, 40, 40, 96, 32, "falling"),
])
def test_error_within_the_arithmetic(cuda, flush, prefix, seqs, heads, kv_heads, dim, bs, order):
    from pagedkv_fusion import ops
    p = accuracy_problem(prefix, seqs, heads, kv_heads, dim, bs, order)
    got = ops.shared_prefix_attention(**p)
    assert cuda.read_device_error() == 0
    want = exact(p)
    err = (got.double() - want).square().mean((0, 2)) / want.square().mean((0, 2))  # of each head
    assert float(err.max().sqrt()) <= LIMIT[flush], float(err.max().sqrt())
