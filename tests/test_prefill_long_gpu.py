"""prefill_attention over long key ranges, V of one sign: the sums' error.

The tensor cores add 16 keys a step and cut, of the sum and of each of the 16
products, what lies two places below the last of the largest: in the mean at
most 16/8 + 1/2 places of 2^-23 of the sum (0.7 places as a part of it).  A sum of
one sign that grows evenly over F tiles of 128 keys (8 steps) loses

  8 F / 2 * 2.5 * 0.7 * 2^-23 = F * 8.4e-7

of itself in the mean, and twice that at most where it does not grow, and O
is added to a sum rounded to nearest every F = 128 tiles.  Beside that an output is rounded to 16 bits, off by eps/2 of its value, and P
by as much for each key, averaged over the keys that carry the weight: 6 standard
deviations, 6 eps/2 / sqrt(3 n), are below eps/8 from n = 100 keys on... the tests
have 300 and more.
"""

from __future__ import annotations

import math

import pytest
import torch

from test_prefill_gpu import DT, cumulative

pytestmark = pytest.mark.gpu


CUT = 128 * 8.4e-7


def problem(seed, n, m, heads, kv_heads, dim, dtype, growth=0.0, spread=2.0):
    """Scores of standard deviation `spread`, rising by `growth` over the keys."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randn(n, heads, dim, generator=g, device="cuda")
    k = torch.randn(m, kv_heads, dim, generator=g, device="cuda") * spread
    q[..., 0] = math.sqrt(dim)
    k[..., 0] = torch.linspace(0, growth, m, device="cuda")[:, None]
    v = (torch.randn(m, kv_heads, dim, generator=g, device="cuda").abs() + 0.5) * \
        (1 + torch.rand(dim, generator=g, device="cuda"))
    return q.to(DT[dtype]), k.to(DT[dtype]), v.to(DT[dtype])


def exact(q, k, v, scale, rows):
    """The definition in 64 bits for the tokens `rows`, and how many keys carry
    each output's weight, 1 / sum w^2."""
    n, m, group = len(q), len(k), q.shape[1] // k.shape[1]
    out = torch.empty(len(rows), q.shape[1], q.shape[2], dtype=torch.float64, device="cuda")
    keys = torch.empty(len(rows), q.shape[1], dtype=torch.float64, device="cuda")
    hidden = torch.arange(m, device="cuda") > (rows + m - n)[:, None]
    for h in range(q.shape[1]):
        s = q[rows, h].double() @ k[:, h // group].double().T * scale
        w = torch.softmax(s.masked_fill_(hidden, -math.inf), 1)
        out[:, h], keys[:, h] = w @ v[:, h // group].double(), 1 / w.square().sum(1)
    return out, keys


def check(q, k, v, rows=None):
    from pagedkv_fusion import _C, ops
    scale = q.shape[2] ** -0.5
    out = ops.prefill_attention(q, k, v, cumulative([len(q)]), scale, cu_seqlens_k=cumulative([len(k)]))
    assert _C.read_device_error() == 0
    rows = torch.arange(len(q), device="cuda") if rows is None else rows
    want, keys = exact(q, k, v, scale, rows)
    got, eps = out[rows].double(), torch.finfo(q.dtype).eps / 2
    averaged = (6 / (3 * keys).sqrt()).clamp(max=1)[..., None]
    tol = want * (eps + eps * averaged + 2 * CUT + 2e-5)
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float(((got - want) / want).abs().max()))
    return out, got, want


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("m", [8192, 20000, 131072, 262144])
def test_sums_of_one_sign_keep_their_size(cuda, dtype, dim, m):
    """The mean error stays that of one stretch of F tiles, however many follow.
    (Against the rounded result, which has the same rounding: what is left of it in
    the mean over 32,768 or 16,384 outputs is under eps/50.)"""
    q, k, v = problem(m + dim, 64, m, 4, 1, dim, dtype)
    _, got, want = check(q, k, v)
    mean = float(((got - want.to(q.dtype).double()) / want).mean())
    assert abs(mean) <= CUT + torch.finfo(q.dtype).eps / 100, mean


@pytest.mark.parametrize("n,m,heads,kv_heads,dim", [
    (600, 17000, 32, 8, 128),    # two row tiles an item, more items than SMs
    (600, 17000, 32, 8, 64),
    (777, 16385, 14, 2, 80),     # groups of 7; one key behind the 128th tile
    (300, 33000, 8, 8, 96),
    (20000, 20000, 4, 2, 128),   # a whole prompt: its last items are long
    (5000, 19000, 16, 4, 32),
])
@pytest.mark.parametrize("growth", [0.0, 10.0, -10.0])
def test_long_ranges(cuda, n, m, heads, kv_heads, dim, growth):
    """Maxima that move before and after O is taken, and fall."""
    q, k, v = problem(n + m, n, m, heads, kv_heads, dim, "f16", growth, spread=1.0)
    g = torch.Generator(device="cuda").manual_seed(1)
    rows = torch.randperm(n, generator=g, device="cuda")[:200]
    rows = torch.cat([rows[rows + m - n >= 4000], torch.tensor([n - 1], device="cuda")])
    out, _, _ = check(q, k, v, rows)
    from pagedkv_fusion import ops
    again = ops.prefill_attention(q, k, v, cumulative([n]), dim ** -0.5, cu_seqlens_k=cumulative([m]))
    assert torch.equal(out, again)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_denominators_and_no_mask(cuda, dim, causal):
    """lse of long rows: the scores' error and the sums' as for short ones."""
    from pagedkv_fusion import ops
    n, m = 150, 20001
    q, k, v = problem(dim, n, m, 4, 2, dim, "bf16")
    scale = dim ** -0.5
    out, lse = ops.prefill_attention(q, k, v, cumulative([n]), scale, cu_seqlens_k=cumulative([m]),
                                     causal=causal, return_lse=True)
    assert cuda.read_device_error() == 0
    hidden = torch.arange(m, device="cuda") > (torch.arange(n, device="cuda") + (m - n if causal else m))[:, None]
    for h in range(4):
        s = (q[:, h].double() @ k[:, h // 2].double().T * scale).masked_fill_(hidden, -math.inf)
        want = torch.softmax(s, 1) @ v[:, h // 2].double()
        assert bool(((out[:, h].double() - want).abs() <= want * (2 ** -8 + 2 * CUT + 2 ** -8)).all())
        ref = torch.logsumexp(s, 1)
        assert bool(((lse[:, h].double() - ref).abs() <= 2e-4 + 2.0 ** -20 * ref.abs()).all())


def test_sequences_of_a_batch_and_nonfinite_values(cuda):
    """Long and short sequences packed give what each gives alone; a NaN stays in
    its rows."""
    from pagedkv_fusion import ops
    lens, ends = [70, 1, 300, 40], [20000, 1, 300, 18000]
    q, k, v = problem(5, sum(lens), sum(ends), 8, 2, 128, "bf16")
    got = ops.prefill_attention(q, k, v, cumulative(lens), 0.1, cu_seqlens_k=cumulative(ends))
    a = b = 0
    for n, m in zip(lens, ends):
        one = ops.prefill_attention(q[a:a + n], k[b:b + m], v[b:b + m], cumulative([n]), 0.1,
                                    cu_seqlens_k=cumulative([m]))
        assert torch.equal(got[a:a + n], one)
        a, b = a + n, b + m
    k[100, 0] = float("nan")
    bad = ops.prefill_attention(q, k, v, cumulative(lens), 0.1, cu_seqlens_k=cumulative(ends))
    assert bool(bad[:70, :4].isnan().all())
    bad[:70, :4] = got[:70, :4]
    assert torch.equal(bad, got)
    assert cuda.read_device_error() == 0


def test_two_graphs_at_once(cuda):
    """Workspaces of two captured calls do not mix, replayed on two streams."""
    from pagedkv_fusion import ops
    graphs, state = [], []
    for seed in (1, 2):
        q, k, v = problem(seed, 200, 20000, 8, 4, 128, "f16")
        cu, ck = cumulative([200]), cumulative([20000])
        ops.prefill_attention(q, k, v, cu, 0.1, cu_seqlens_k=ck)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = ops.prefill_attention(q, k, v, cu, 0.1, cu_seqlens_k=ck)
        graphs.append(gr)
        state.append((q, k, v, cu, ck, out))
    for _ in range(3):
        for s in state:
            s[0].normal_()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for st, gr in zip(streams, graphs):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for q, k, v, cu, ck, out in state:
            assert torch.equal(out, ops.prefill_attention(q, k, v, cu, 0.1, cu_seqlens_k=ck))
    assert cuda.read_device_error() == 0
