"""shared_prefix_attention against softmax attention in 64 bits over the
dequantized [prefix | own] tokens, and against quant_paged_attention over the
joined tables.

Tolerance, per output, with A = sum_j softmax_j |v_j|, S = |scale| sum_d |q_d k_d|
(largest over the row's tokens), D channels, n tokens: a query is kept to 2^-22
of its values, a score is a sum of 2 D products in fp32 (2^-23 each), an
exponential and a probability are kept to 2^-21, sums run over n tokens:

  |got - want| <= A (2 (2 D + 2) 2^-23 S + 2 n 2^-23 + 2^-19) + floor

Relative steps end where fixed point begins: p * v_scale of the prefix is two
fp16 numbers whose smallest step is 2^-24, with the part's largest p at 2^13 or
more and v_scale relative to the largest, so a token is off by up to half a
step, 2^-25 / 2^13 of the largest weight w times the largest value; the decode
kernel's own tokens have 24-bit fixed point, half a step 2^-25 of theirs:

  floor = 2^-38 n0 max(w0) max|v0| + 2^-25 n1 max(w1) max|v1|

(0: prefix, 1: own tokens; max|v| is the largest scale times 127).
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def problem(seed, prefix, lens, heads, kv_heads, dim, bs, wide=0, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    shared = -(-prefix // bs)
    pages = [-(-n // bs) for n in lens]
    nb = shared + sum(pages) + 2
    perm = torch.randperm(nb, generator=g, device="cuda").to(torch.int32)
    width = max(pages, default=0) + wide
    tables = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    at = shared
    for i, n in enumerate(pages):
        tables[i, :n] = perm[at:at + n]
        at += n
    shape = (nb, bs, kv_heads, dim)
    codes = [torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8) for _ in "kv"]
    scales = [torch.exp(spread * torch.randn(nb, kv_heads, generator=g, device="cuda")) / 60
              for _ in "kv"]
    q = torch.randn(len(lens), heads, dim, generator=g, device="cuda")
    return dict(q=q, k_cache_q=codes[0], k_scale=scales[0], v_cache_q=codes[1], v_scale=scales[1],
                prefix_table=torch.cat([perm[:shared], perm[:wide]]),
                prefix_len=torch.tensor([prefix], dtype=torch.int32, device="cuda"),
                block_tables=tables, seq_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                sm_scale=1.0 / math.sqrt(dim))


def reference(p):
    q = p["q"].double()
    bs, kv = p["k_cache_q"].shape[1:3]
    group, D = q.shape[1] // kv, q.shape[2]
    want, tol = torch.zeros_like(q), torch.zeros_like(q)
    n0 = int(p["prefix_len"])

    def tokens(cache, scale, pages, n, h):
        x = cache[pages.long(), :, h].double() * scale[pages.long(), h].double()[:, None, None]
        return x.flatten(0, 1)[:n]

    for h in range(kv):
        front = [tokens(p[c], p[s], p["prefix_table"][:-(-n0 // bs)], n0, h)
                 for c, s in (("k_cache_q", "k_scale"), ("v_cache_q", "v_scale"))]
        for i, n in enumerate(p["seq_lens"].tolist()):
            if n + n0 == 0:
                continue
            pages = p["block_tables"][i, :-(-n // bs)]
            k = torch.cat([front[0], tokens(p["k_cache_q"], p["k_scale"], pages, n, h)])
            v = torch.cat([front[1], tokens(p["v_cache_q"], p["v_scale"], pages, n, h)])
            qh = q[i, h * group:(h + 1) * group]
            w = torch.softmax(qh @ k.T * p["sm_scale"], 1)
            S = (qh.abs() @ k.abs().T * abs(p["sm_scale"])).amax(1, keepdim=True)
            want[i, h * group:(h + 1) * group] = w @ v
            floor = 0.0
            for part, m, sc, step in ((slice(0, n0), n0, p["prefix_table"][:-(-n0 // bs)], 2.0 ** -38),
                                      (slice(n0, None), n, pages, 2.0 ** -25)):
                if m:
                    most = 127 * p["v_scale"][sc.long(), h].double().abs().max()
                    floor = floor + step * m * w[:, part].amax(1, keepdim=True) * most
            tol[i, h * group:(h + 1) * group] = floor + (w @ v.abs()) * (
                2 * (2 * D + 2) * 2.0 ** -23 * S + 2 * (n + n0) * 2.0 ** -23 + 2.0 ** -19)
    return want, tol


def check(p, error=0):
    from pagedkv_fusion import _C, ops
    out = ops.shared_prefix_attention(**p)
    assert _C.read_device_error() == error
    want, tol = reference(p)
    assert out.dtype == torch.float32 and out.is_contiguous()
    bad = ~((out.double() - want).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float((out - want).abs().max()), bad.nonzero()[:5].tolist())
    assert torch.equal(out, ops.shared_prefix_attention(**p))  # the same bits every time
    return out


@pytest.mark.parametrize("prefix,lens,heads,kv_heads,dim,bs", [
    (1, [0], 1, 1, 128, 16),
    (512, [1, 2, 3, 5, 8, 13, 21, 32], 8, 8, 128, 16),
    (129, [7, 0, 100], 32, 8, 128, 16),          # a page ends inside the second tile
    (1000, [17] * 70, 8, 2, 128, 16),            # 280 rows: two pairs of row tiles
    (777, [5, 300, 64, 1], 16, 2, 128, 32),
    (2040, [33] * 32, 32, 8, 128, 16),           # exactly one row tile
    (2040, [33] * 33, 32, 8, 128, 16),
    (640, [9, 20], 6, 2, 96, 16),                # groups of 3
    (333, [40, 1], 14, 2, 64, 16),               # groups of 7
    (333, [40, 1], 4, 4, 32, 8),
    (100, [3, 50], 20, 1, 64, 24),               # pages that do not divide a tile
    (5000, [1000, 10], 8, 1, 128, 64),
    (20000, [12] * 3, 4, 1, 128, 16),            # many parts
    (0, [5, 0, 60], 8, 2, 128, 16),              # no prefix at all
    (250, [0, 0, 0], 8, 2, 128, 16),             # and nothing else
])
def test_matches_reference(cuda, prefix, lens, heads, kv_heads, dim, bs):
    check(problem(prefix + dim, prefix, lens, heads, kv_heads, dim, bs))


@pytest.mark.parametrize("prefix,lens,heads,dim,bs", [
    (6000, [9, 1], 40, 128, 16),       # 2 rows of a KV head: most warps have none
    (6000, [9, 1, 0], 40, 64, 16),
    (4990, [3] * 40, 40, 128, 16),     # 40 rows: a warp and a part of one
    (4990, [3] * 70, 40, 96, 24),
    (4500, [1] * 130, 40, 128, 16),    # a row and a half tile: sums beside O in memory
    (4500, [1] * 130, 40, 64, 32),
])
def test_parts_of_many_tiles(cuda, prefix, lens, heads, dim, bs):
    """Many KV heads leave each CTA 12 to 16 tiles of the prefix."""
    check(problem(prefix + dim, prefix, lens, heads, heads, dim, bs))


@pytest.mark.parametrize("prefix,lens,heads,kv_heads,dim,bs,wide", [
    (40, [3000, 64, 65, 0, 1, 63], 12, 4, 96, 16, 2000),  # parts of more than 64 tokens
    (0, [1000, 5, 128], 22, 2, 128, 16, 0),               # 11 heads: a group in two parts
    (16, [700, 300], 5, 5, 32, 8, 3000),
    (50, [200, 49, 48], 16, 2, 64, 24, 5),                # 48 tokens of 2 pages at a time
    (50, [200, 64], 3, 3, 64, 64, 0),
])
def test_own_tokens_of_any_shape(cuda, prefix, lens, heads, kv_heads, dim, bs, wide):
    from pagedkv_fusion import _C, ops
    p = problem(prefix + dim, prefix, lens, heads, kv_heads, dim, bs, wide=wide)
    want = check(p)
    for bad in (float("nan"), float("inf")):
        q = p["q"].clone()
        q[1, heads - 1] = bad
        out = ops.shared_prefix_attention(**dict(p, q=q))
        assert bool((~out[1, heads - 1].isfinite()).all())
        out[1, heads - 1] = want[1, heads - 1]
        assert torch.equal(out, want)
    # tokens on a page outside the cache do not count, nor those past the table
    tables = p["block_tables"].clone()
    tables[0, 1] = p["k_cache_q"].shape[0]
    out = ops.shared_prefix_attention(**dict(p, block_tables=tables))
    assert _C.read_device_error() == 1
    kept = dict(p, block_tables=p["block_tables"].clone(), seq_lens=p["seq_lens"].clone())
    kept["block_tables"][0, 1:-1] = p["block_tables"][0, 2:]
    kept["seq_lens"][0] -= bs
    again, tol = reference(kept)
    assert bool(((out[0].double() - again[0]).abs() <= tol[0]).all())
    lens = p["seq_lens"].clone()
    lens[0] = p["block_tables"].shape[1] * bs + 1
    full = dict(p, block_tables=p["block_tables"].clamp(min=0))
    out = ops.shared_prefix_attention(**dict(full, seq_lens=lens))
    assert _C.read_device_error() == 4
    lens[0] -= 1
    assert torch.equal(out, ops.shared_prefix_attention(**dict(full, seq_lens=lens)))


@pytest.mark.parametrize("prefix,heads,kv_heads,bs", [(1024, 8, 8, 16), (320, 32, 8, 16),
                                                      (96, 8, 2, 32)])
def test_agrees_with_decode_over_joined_tables(cuda, prefix, heads, kv_heads, bs):
    from pagedkv_fusion import ops
    p = problem(3, prefix, [10, 333, 64, 1, 0], heads, kv_heads, 128, bs)
    out = check(p)
    n = prefix // bs
    tables = torch.cat([p["prefix_table"][:n].expand(5, n), p["block_tables"]], 1)
    want = ops.quant_paged_attention(p["q"], p["k_cache_q"], p["k_scale"], p["v_cache_q"], p["v_scale"],
                                     tables, p["seq_lens"] + prefix, p["sm_scale"])
    np.testing.assert_allclose(out.cpu().numpy(), want.cpu().numpy(), rtol=2e-4, atol=2e-4)


def test_score_ranges_and_signs(cuda):
    """Queries of any magnitude, a negative scale, scales of very different
    pages, maxima that grow from tile to tile."""
    p = problem(7, 900, [40, 3, 0], 8, 2, 128, 16, spread=3.0)
    check(p)
    check(dict(p, sm_scale=-0.05))
    check(dict(p, sm_scale=0.0))
    check(dict(p, q=p["q"] * 1e-30))
    check(dict(p, q=torch.zeros_like(p["q"])))
    check(dict(p, q=p["q"] * 1e30, sm_scale=p["sm_scale"] * 1e-30))
    ramp = p["k_scale"].clone()
    ramp[p["prefix_table"].long()] = torch.linspace(1e-3, 0.3, len(p["prefix_table"]),
                                                    device="cuda")[:, None]
    check(dict(p, k_scale=ramp))
    zero = torch.zeros_like(p["v_scale"])
    assert bool((check(dict(p, v_scale=zero)) == 0).all())


def test_rows_do_not_touch_each_other(cuda):
    """A sequence with non-finite queries leaves the others' bits alone."""
    from pagedkv_fusion import ops
    p = problem(8, 500, [40, 3, 0, 77], 8, 2, 128, 16)
    want = ops.shared_prefix_attention(**p)
    for bad in (float("nan"), float("inf")):
        q = p["q"].clone()
        q[1] = bad
        out = ops.shared_prefix_attention(**dict(p, q=q))
        assert bool((~out[1].isfinite()).all())
        assert torch.equal(out[[0, 2, 3]], want[[0, 2, 3]])


def test_stale_pages_behind_the_end_are_not_read(cuda):
    """Scales of pages that no token reaches may be anything."""
    from pagedkv_fusion import ops
    p = problem(9, 100, [40, 3], 8, 2, 128, 16, wide=3)
    want = check(p)
    unused = torch.ones(len(p["k_scale"]), dtype=torch.bool, device="cuda")
    unused[p["prefix_table"][:7].long()] = False
    for i, n in enumerate((3, 1)):
        unused[p["block_tables"][i, :n].long()] = False
    ks, vs = p["k_scale"].clone(), p["v_scale"].clone()
    ks[unused], vs[unused] = float("nan"), float("inf")
    table = p["prefix_table"].clone()
    table[7:] = 10 ** 6
    assert torch.equal(ops.shared_prefix_attention(**dict(p, k_scale=ks, v_scale=vs, prefix_table=table)),
                       want)
    assert cuda.read_device_error() == 0


def test_bad_tables_and_lengths(cuda):
    from pagedkv_fusion import ops
    p = problem(10, 160, [20, 5], 8, 2, 128, 16)
    for bad in (-1, 10 ** 6):
        table = p["prefix_table"].clone()
        table[3] = bad
        out = ops.shared_prefix_attention(**dict(p, prefix_table=table))
        assert cuda.read_device_error() == 1
        keep = [i for i in range(10) if i != 3]     # the page's tokens are left out
        want, tol = reference(dict(p, prefix_table=p["prefix_table"][keep],
                                   prefix_len=torch.tensor([144], device="cuda")))
        assert bool(((out.double() - want).abs() <= tol).all())
    out = ops.shared_prefix_attention(**dict(p, prefix_len=torch.tensor([500], device="cuda")))
    assert cuda.read_device_error() == 4
    assert torch.equal(out, ops.shared_prefix_attention(**p))
    ops.shared_prefix_attention(**dict(p, seq_lens=torch.tensor([20, 50], device="cuda")))
    assert cuda.read_device_error() == 4
    none = ops.shared_prefix_attention(**dict(p, prefix_len=torch.tensor([-3], device="cuda"),
                                              seq_lens=torch.tensor([0, -1], device="cuda")))
    assert bool((none == 0).all()) and cuda.read_device_error() == 0


def test_large_cache_offsets(cuda):
    """Pages beyond 2^31 bytes of the cache."""
    nb, hkv = 140000, 8
    g = torch.Generator(device="cuda").manual_seed(1)
    cache = torch.randint(-127, 128, (nb, 16, hkv, 128), generator=g, device="cuda", dtype=torch.int8)
    scale = torch.rand(nb, hkv, generator=g, device="cuda") / 100
    last = torch.arange(nb - 40, nb, device="cuda", dtype=torch.int32)
    check(dict(q=torch.randn(3, 8, 128, generator=g, device="cuda"), k_cache_q=cache, k_scale=scale,
               v_cache_q=cache, v_scale=scale, prefix_table=last[:30],
               prefix_len=torch.tensor([475], device="cuda"), block_tables=last[30:36].view(3, 2),
               seq_lens=torch.tensor([20, 32, 1], device="cuda"), sm_scale=0.1))


def test_graph_follows_lengths_and_workspaces_do_not_mix(cuda):
    """Two captured calls replayed at once on two streams, with new queries,
    prefix lengths and own lengths."""
    from pagedkv_fusion import ops
    graphs, state = [], []
    for seed in (1, 2):
        p = problem(seed, 700, [90, 90, 90], 8, 2, 128, 16)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops.shared_prefix_attention(**p)
        torch.cuda.current_stream().wait_stream(side)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = ops.shared_prefix_attention(**p)
        graphs.append(gr)
        state.append((p, out))
    for lens, n in (([1, 0, 90], 700), ([40, 90, 16], 3), ([0, 0, 0], 0), ([5, 6, 7], 640)):
        for p, _ in state:
            p["q"].normal_()
            p["seq_lens"].copy_(torch.tensor(lens))
            p["prefix_len"].fill_(n)
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for st, gr in zip(streams, graphs):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for p, out in state:
            assert torch.equal(out, ops.shared_prefix_attention(**p))
    assert cuda.read_device_error() == 0


def test_copies_of_odd_inputs_and_host_inputs(cuda):
    from pagedkv_fusion import ops
    p = problem(12, 100, [9, 30], 4, 2, 64, 16)
    want = ops.shared_prefix_attention(**p)
    flat = torch.empty(p["q"].numel() + 1, device="cuda")
    flat[1:] = p["q"].flatten()
    cut = torch.empty(p["k_cache_q"].numel() + 1, dtype=torch.int8, device="cuda")
    cut[1:] = p["k_cache_q"].flatten()
    odd = dict(p, q=flat[1:].view(p["q"].shape), k_cache_q=cut[1:].view(p["k_cache_q"].shape),
               seq_lens=p["seq_lens"].long(), block_tables=p["block_tables"].t().contiguous().t())
    assert torch.equal(ops.shared_prefix_attention(**odd), want)
    host = {k: v.cpu().numpy() if isinstance(v, torch.Tensor) else v for k, v in p.items()}
    got = ops.shared_prefix_attention(**host)
    assert isinstance(got, np.ndarray)
    np.testing.assert_array_equal(got, want.cpu().numpy())
    empty = dict(p, q=p["q"][:0], block_tables=p["block_tables"][:0], seq_lens=p["seq_lens"][:0])
    assert ops.shared_prefix_attention(**empty).shape == (0, 4, 64)


def test_refusals(cuda):
    from pagedkv_fusion import ops
    p = problem(13, 100, [9, 30], 4, 2, 64, 16)
    for kw, msg in [
        (dict(q=p["q"].half()), "float32"), (dict(k_cache_q=p["k_cache_q"].float()), "int8"),
        (dict(k_scale=p["k_scale"][:, :1]), "scales"), (dict(prefix_table=p["prefix_table"].long()), "int32"),
        (dict(prefix_table=p["block_tables"]), "expected"), (dict(block_tables=p["block_tables"][:1]), "rows"),
        (dict(prefix_len=torch.tensor([3, 4], device="cuda")), "prefix_len"),
        (dict(prefix_len=torch.tensor([3.0], device="cuda")), "prefix_len"),
        (dict(q=p["q"][:, :3]), "GQA"), (dict(q=p["q"].clone().requires_grad_()), "backward"),
    ]:
        with pytest.raises(RuntimeError, match=msg):
            ops.shared_prefix_attention(**dict(p, **kw))
    big = problem(14, 10, [3], 2, 2, 160, 16)
    with pytest.raises(RuntimeError, match="head_dim"):
        ops.shared_prefix_attention(**big)
