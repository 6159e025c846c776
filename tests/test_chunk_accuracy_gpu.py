"""chunk_attention held to the accuracy that it is built for: its errors within the limits of the
arithmetic (derived, and shown to tell a loss of precision, in test_chunk_accuracy_cpu.py).
"""

from __future__ import annotations

import math

import pytest
import torch

from test_chunk_accuracy_cpu import LIMIT, SCORE_LIMIT, SPREAD

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def accuracy_problem(q_lens, keys, heads, kv_heads, dim, bs, dtype="f32", order="mixed"):
    """Sequences over the same pages, V codes of one sign, the pages' K scales uneven, or rising or
    falling along them."""
    g = torch.Generator(device="cuda").manual_seed(keys + len(q_lens))
    n, S = -(-keys // bs), len(q_lens)
    table = torch.randperm(n + 2, generator=g, device="cuda")[:n].to(torch.int32)
    k_scale, v_scale = (0.5 + torch.rand(n + 2, kv_heads, generator=g, device="cuda") for _ in "kv")
    if order != "mixed":
        ramp = torch.linspace(0.1, 1.5, n, device="cuda")[:, None]
        k_scale[table.long()] = ramp if order == "rising" else ramp.flip(0)
    shape = (n + 2, bs, kv_heads, dim)
    return dict(
        q=torch.randn(sum(q_lens), heads, dim, generator=g, device="cuda").to(TYPES[dtype]),
        k_cache_q=torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8),
        k_scale=k_scale * SPREAD / 73.3,
        v_cache_q=torch.randint(1, 128, shape, generator=g, device="cuda", dtype=torch.int8),
        v_scale=v_scale / 64, block_tables=table.expand(S, -1).contiguous(),
        seq_lens=torch.full((S,), keys, dtype=torch.int32, device="cuda"),
        cu_seqlens=torch.tensor([0] + q_lens, device="cuda").cumsum(0).to(torch.int32), sm_scale=dim ** -0.5)


def exact(p):
    """Outputs, log denominators and gathered weights of the keys, in 64 bits."""
    q, table = p["q"].double(), p["block_tables"][0].long()
    kv, n = p["k_scale"].shape[1], int(p["seq_lens"][0])
    group = q.shape[1] // kv
    out, lse, weights = torch.zeros_like(q), q.new_zeros(q.shape[:2]), q.new_zeros(n)
    counts = p["cu_seqlens"].diff().tolist()
    last = torch.cat([torch.arange(n - c, n, device="cuda") for c in counts])
    seen = torch.arange(n, device="cuda") <= last[:, None]
    for h in range(kv):
        k, v = ((p[c][table, :, h].double() * p[s][table, h].double()[:, None, None]).flatten(0, 1)[:n]
                for c, s in (("k_cache_q", "k_scale"), ("v_cache_q", "v_scale")))
        for a in range(h * group, (h + 1) * group):
            s = torch.where(seen, q[:, a] @ k.T * p["sm_scale"], -math.inf)
            lse[:, a] = torch.logsumexp(s, 1)
            w = torch.softmax(s, 1)
            out[:, a] = w @ v
            weights += w.sum(0) / q.shape[1]
    return out, lse, weights


def error(got, want):
    return float(((got.double() - want).square().mean() / want.square().mean()).sqrt())


SHAPES = [
    # few rows: a warp has the whole of a sequence, or a part that a few or many join
    ([1] * 60, 32768, 40, 40, 64, 16, "mixed"), ([1] * 60, 32768, 40, 40, 128, 16, "falling"),
    ([1] * 60, 4096, 40, 40, 128, 16, "rising"), ([1] * 4, 4096, 8, 8, 128, 16, "mixed"),
    ([4, 1], 20000, 8, 2, 128, 16, "mixed"), ([1] * 64, 16384, 40, 40, 128, 24, "falling"),
    ([1] * 32, 20000, 40, 40, 256, 16, "falling"), ([40], 16384, 8, 4, 256, 16, "mixed"),
    # many: parts of up to 55 tiles, pairs of row tiles, or even and odd key tiles apart
    ([256], 16384, 8, 2, 128, 16, "mixed"), ([1024], 32768, 8, 8, 128, 16, "falling"),
    ([1024], 32768, 8, 8, 64, 16, "rising"), ([40], 32768, 40, 40, 96, 32, "mixed"),
]


@pytest.mark.parametrize("q_lens,keys,heads,kv_heads,dim,bs,order", SHAPES)
def test_error_within_the_arithmetic(cuda, q_lens, keys, heads, kv_heads, dim, bs, order):
    from pagedkv_fusion import ops
    p = accuracy_problem(q_lens, keys, heads, kv_heads, dim, bs, order=order)
    out, lse = ops.chunk_attention(**p, return_lse=True)
    assert cuda.read_device_error() == 0
    want, want_lse, _ = exact(p)
    err = (out.double() - want).square().mean((0, 2)) / want.square().mean((0, 2))  # of each head
    assert float(err.max().sqrt()) <= LIMIT, float(err.max().sqrt())
    off = float((lse.double() - want_lse).square().mean().sqrt())
    assert off <= SCORE_LIMIT[max(dim, 128)], off


@pytest.mark.parametrize("q_lens,keys,heads,kv_heads,dim,bs", [
    ([1] * 60, 32768, 40, 40, 128, 16), ([1] * 60, 32768, 40, 40, 64, 24), ([1024], 32768, 8, 8, 128, 16)])
def test_mean_of_16_bit_results(cuda, q_lens, keys, heads, kv_heads, dim, bs):
    """Roundings to 16 bits have either sign and leave the mean over all results; what the sums
    lose does not: 1.2 / 2 * 0.7 * 2^-23 for 16 keys (see above), of 16,384 at most 5.2e-5."""
    from pagedkv_fusion import ops
    p = accuracy_problem(q_lens, keys, heads, kv_heads, dim, bs, "f16")
    want = exact(p)[0]
    mean = float((ops.chunk_attention(**p).double() - want).mean() / want.mean())
    assert abs(mean) <= 6e-5, mean


@pytest.mark.parametrize("dtype,q_lens,keys,heads,kv_heads,dim,bs,more", [
    # few rows: P as two fp16 numbers for fp16 results, as one for bf16 ones
    ("f16", [1] * 60, 4096, 40, 40, 128, 16, 1.03), ("f16", [4, 1, 8], 3000, 32, 8, 64, 24, 1.03),
    ("f16", [1, 3], 5000, 8, 2, 256, 16, 1.03),
    ("bf16", [1] * 60, 4096, 40, 40, 128, 16, 1.015), ("bf16", [4, 1, 8], 3000, 32, 8, 64, 24, 1.015),
    # many: one number
    ("f16", [512], 4096, 8, 2, 128, 16, 1.5), ("bf16", [512], 4096, 8, 2, 128, 16, 1.015),
])
def test_error_beside_the_rounding_of_results(cuda, dtype, q_lens, keys, heads, kv_heads, dim, bs, more):
    """V of either sign: the error is at most `more` times what rounding the exact result leaves.
    A rounding of P to fp16 is like the result's own to fp16 (sqrt(2) of it together) and an eighth
    of one to bf16 (1.008)."""
    from pagedkv_fusion import ops
    p = accuracy_problem(q_lens, keys, heads, kv_heads, dim, bs, dtype)
    p["v_cache_q"].random_(-127, 128)
    want = exact(p)[0]
    assert error(ops.chunk_attention(**p), want) <= more * error(want.to(p["q"].dtype), want)
