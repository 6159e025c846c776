"""prefill_attention against softmax attention in 64 bits.

Tolerance, per output: P is rounded to the inputs' type (half a step each) and
so is the output; the scores are fp32 sums of D products (at most D roundings
of 2^-24 of the sum of magnitudes), the exponential's approximation and the
sums over n keys are fp32:

  |got - want| <= eps/2 (A + |want|) + A (2 D 2^-24 S + 2 n 2^-24 + 2^-20) + sub

with A = sum_j softmax_j |v_j|, S = scale sum_d |q_d k_d| (its largest over the
row's keys), and sub = 2^-25 sum_j |v_j| for fp16, whose probabilities below
2^-14 are subnormal (the denominator is at least 1).
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def cumulative(lens):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")


def reference(q, k, v, q_lens, k_lens, scale, causal, heads=None):
    """(want, lse, tolerance) in float64; rows behind the last sequence are zero."""
    dt, D = q.dtype, q.shape[2]
    q, k, v = q.double(), k.double(), v.double()
    group = q.shape[1] // k.shape[1]
    want, tol = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    q0 = k0 = 0
    eps = torch.finfo(dt).eps / 2
    for n, m in zip(q_lens, k_lens):
        seen = torch.ones(n, m, dtype=torch.bool, device="cuda")
        if causal:
            seen = seen.tril(m - n)
        for h in heads if heads is not None else range(q.shape[1]):
            qs, ks, vs = q[q0:q0 + n, h], k[k0:k0 + m, h // group], v[k0:k0 + m, h // group]
            s = torch.where(seen, qs @ ks.T * scale, -math.inf)
            row = s.amax(1, keepdim=True) if m else torch.zeros(n, 1, device="cuda", dtype=q.dtype)
            e = torch.where(seen, torch.exp(s - row.clamp(min=-1e300)), 0.0)
            den = e.sum(1, keepdim=True)
            p = e / den.clamp(min=1e-300)
            w = p @ vs
            A = p @ vs.abs()
            S = (torch.where(seen, qs.abs() @ ks.abs().T, 0.0) * scale).amax(1, keepdim=True) if m else 0
            want[q0:q0 + n, h] = w
            lse[q0:q0 + n, h] = torch.where(den > 0, torch.log(den) + row, -math.inf)[:, 0]
            t = eps * (A + w.abs()) + A * (2 * D * 2.0 ** -24 * S + 2 * m * 2.0 ** -24 + 2.0 ** -20)
            if dt == torch.float16:
                t = t + 2.0 ** -25 * (seen.double() @ vs.abs()) + 2.0 ** -25
            tol[q0:q0 + n, h] = t
        q0, k0 = q0 + n, k0 + m
    return want, lse, tol


def check(q, k, v, q_lens, k_lens, causal=True, scale=None, heads=None):
    from pagedkv_fusion import _C, ops
    scale = scale or 1.0 / math.sqrt(q.shape[2])
    cq, ck = cumulative(q_lens), cumulative(k_lens)
    out, lse = ops.prefill_attention(q, k, v, cq, scale, cu_seqlens_k=ck, causal=causal, return_lse=True)
    assert _C.read_device_error() == 0
    want, wlse, tol = reference(q, k, v, q_lens, k_lens, scale, causal, heads)
    assert out.dtype == q.dtype and out.shape == q.shape and out.is_contiguous()
    pick = slice(None) if heads is None else heads
    o, w, t = out[:, pick].double(), want[:, pick], tol[:, pick]
    bad = ~((o - w).abs() <= t)
    assert not bool(bad.any()), (int(bad.sum()), float((o - w).abs().max()), bad.nonzero()[:5].tolist())
    finite = wlse[:, pick] > -math.inf
    assert torch.equal(lse[:, pick] > -math.inf, finite)
    # lse: score error as above, the sum's and the logarithm's roundings
    err = (lse[:, pick].double() - wlse[:, pick])[finite].abs()
    assert bool((err <= 2e-4 + 2.0 ** -20 * wlse[:, pick][finite].abs()).all()), float(err.max())
    if q_lens == k_lens and heads is None:
        again = ops.prefill_attention(q, k, v, cq, scale, causal=causal)
        assert torch.equal(again, out)  # and the same bits every time
    return out


def problem(seed, q_lens, k_lens, heads, kv_heads, dim, dtype, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(DT[dtype])  # noqa: E731
    return (r(sum(q_lens) + pad, heads, dim), r(sum(k_lens) + pad, kv_heads, dim),
            r(sum(k_lens) + pad, kv_heads, dim))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lens,heads,kv_heads,dim", [
    ([1], 1, 1, 64),
    ([37], 8, 8, 64),
    ([128], 2, 2, 128),
    ([129, 1, 127, 256], 2, 1, 128),
    ([1, 2, 3, 300, 5, 64, 65], 8, 2, 128),
    ([777], 32, 8, 128),
    ([200, 100], 6, 2, 96),        # groups of 3: 42 tokens a row tile
    ([333], 14, 2, 80),            # groups of 7
    ([70, 3], 20, 1, 32),          # groups of 20
    ([19, 140], 128, 1, 64),       # one token a row tile
    ([1500, 20], 4, 4, 8),
    ([40] * 70, 4, 2, 64),         # more sequences than a warp
    ([2100], 4, 1, 128),
])
def test_causal_prompts(cuda, dtype, lens, heads, kv_heads, dim):
    q, k, v = problem(len(lens) + dim, lens, lens, heads, kv_heads, dim, dtype)
    check(q, k, v, lens, lens)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("q_lens,k_lens,causal", [
    ([1], [5000], True),                    # a single new token
    ([100, 3, 64], [612, 3, 1000], True),   # chunks of longer prompts
    ([300], [20], True),                    # most rows see nothing
    ([130, 200], [0, 129], True),           # a sequence without keys
    ([0, 50, 0], [10, 50, 0], True),        # and without tokens
    ([77, 256], [300, 128], False),
    ([5], [0], False),
])
def test_lengths_that_differ(cuda, dtype, q_lens, k_lens, causal):
    q, k, v = problem(sum(k_lens), q_lens, k_lens, 8, 2, 128, dtype)
    check(q, k, v, q_lens, k_lens, causal)


def test_score_ranges(cuda):
    """Rows whose maxima grow tile by tile, and very large and small scores."""
    lens = [700]
    q, k, v = problem(1, lens, lens, 4, 2, 64, "f16")
    ramp = torch.linspace(0.1, 30, 700, device="cuda")[:, None, None]
    check(q, (k * ramp).half(), v, lens, lens, scale=0.5)
    check(q, (k * ramp.flip(0)).half(), v, lens, lens, scale=0.5)
    check((q * 1e-3).half(), k, v, lens, lens, scale=1e-3)
    check(q.abs(), -k.abs(), v, lens, lens, scale=3.0)   # every score far below zero


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_nonfinite_values_stay_where_they_are_seen(cuda, dtype, bad):
    """Non-finite keys and values reach the rows that see them and no others:
    not earlier tokens, not other sequences, nor from rows behind the last."""
    from pagedkv_fusion import ops
    lens = [150, 300, 70]
    q, k, v = problem(5, lens, lens, 8, 2, 128, dtype, pad=40)
    clean = ops.prefill_attention(q, k, v, cumulative(lens), 0.1)
    for t, d in ((149, 3), (150 + 130, 127), (150 + 257, 64), (150 + 299, 0), (450 + 33, 5)):
        v2 = v.clone()
        v2[t, 1, d] = bad
        v2[520:] = bad
        k2 = k.clone()
        k2[520:] = bad
        out = ops.prefill_attention(q, k2, v2, cumulative(lens), 0.1)
        end = 150 if t < 150 else 450 if t < 450 else 520
        hit = torch.zeros_like(out, dtype=torch.bool)
        hit[t:end, 4:, d] = True
        assert torch.equal(~out.isfinite(), hit), (t, d, (~out.isfinite() ^ hit).nonzero()[:5])
        keep = ~hit
        # a tile whose V was cleaned gives the same products
        assert torch.equal(out[keep], clean[keep])
        if bad != bad:
            assert bool(out[hit].isnan().all())
        elif t >= end - 128:  # all its rows are in tiles with masked keys
            assert bool((out[hit] == bad).all())
        assert bool((out[520:] == 0).all())
    k2 = k.clone()
    k2[200, 0] = float("nan")   # a key: the rows that see it are NaN
    out = ops.prefill_attention(q, k2, v, cumulative(lens), 0.1)
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[200:450, :4] = True
    assert torch.equal(out.isnan(), hit)


def test_strided_views(cuda):
    """Views of one projection's output, transposed layouts, misaligned rows."""
    from pagedkv_fusion import ops
    g = torch.Generator(device="cuda").manual_seed(8)
    lens = [90, 41]
    qkv = torch.randn(131, 8 + 2 + 2, 64, generator=g, device="cuda").half()
    q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
    want = ops.prefill_attention(q.contiguous(), k.contiguous(), v.contiguous(), cumulative(lens), 0.2)
    assert torch.equal(ops.prefill_attention(q, k, v, cumulative(lens), 0.2), want)
    heads_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    assert torch.equal(ops.prefill_attention(*heads_first, cumulative(lens), 0.2), want)
    odd = torch.empty(131 * 12 * 64 + 1, device="cuda").half()[1:].view(131, 12, 64)
    odd.copy_(qkv)
    assert torch.equal(ops.prefill_attention(odd[:, :8], odd[:, 8:10], odd[:, 10:], cumulative(lens), 0.2),
                       want)
    one = k[:, :1].expand(131, 4, 64)  # stride 0
    check(q, one, one, lens, lens, scale=0.2)


def test_offsets_past_32_bits(cuda):
    """Keys of more than 2^31 elements; the last tokens of the last heads."""
    m, hkv = 262144, 66
    g = torch.Generator(device="cuda").manual_seed(4)
    k = torch.randn(m, hkv, 128, generator=g, device="cuda", dtype=torch.float16)
    v = torch.randn(m, hkv, 128, generator=g, device="cuda", dtype=torch.float16)
    q = torch.randn(3, hkv, 128, generator=g, device="cuda", dtype=torch.float16)
    k[-2:, -1] = q[-2:, -1]  # the last keys carry most of the weight of the last head
    check(q, k, v, [3], [m], heads=[0, 65])


def test_padded_batch_and_bad_cu_seqlens(cuda):
    from pagedkv_fusion import ops
    q, k, v = problem(2, [100], [100], 4, 2, 64, "bf16", pad=300)
    out, lse = ops.prefill_attention(q, k, v, cumulative([60, 40]), 0.1, return_lse=True)
    assert bool((out[100:] == 0).all()) and bool((lse[100:] == -math.inf).all())
    assert torch.equal(out[:60], ops.prefill_attention(q[:60], k[:60], v[:60], cumulative([60]), 0.1))
    assert cuda.read_device_error() == 0
    for cu in ([0, 50, 30, 100], [0, 500], [-4, 60], [30, 20]):
        ops.prefill_attention(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"), 0.1)
        assert cuda.read_device_error() == 6


def test_stream_and_graph(cuda):
    """Captured once, replayed for new inputs and lengths; two graphs at once."""
    from pagedkv_fusion import ops
    lens = [120, 300]
    graphs, state = [], []
    for seed in (1, 2):
        q, k, v = problem(seed, lens, lens, 8, 2, 128, "bf16")
        cu = cumulative(lens)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            first = ops.prefill_attention(q, k, v, cu, 0.1)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(first, ops.prefill_attention(q, k, v, cu, 0.1))
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = ops.prefill_attention(q, k, v, cu, 0.1)
        graphs.append(gr)
        state.append((q, k, v, cu, out))
    for a, b in (([120, 300], [420, 0]), ([1, 419], [7, 413])):
        for gr, s, ls in zip(graphs, state, (a, b)):
            s[3].copy_(cumulative(ls))
            s[0].normal_()
        s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
        for st, gr in zip((s1, s2), graphs):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for q, k, v, cu, out in state:
            assert torch.equal(out, ops.prefill_attention(q, k, v, cu, 0.1))
    assert cuda.read_device_error() == 0


def test_empty_calls_and_host_inputs(cuda):
    from pagedkv_fusion import ops
    none = torch.zeros(0, 4, 64, device="cuda", dtype=torch.float16)
    out, lse = ops.prefill_attention(none, none, none, cumulative([0, 0]), 0.1, return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    some = torch.ones(5, 4, 64, device="cuda", dtype=torch.float16)
    assert bool((ops.prefill_attention(some, some, some, cumulative([]), 0.1) == 0).all())
    assert bool((ops.prefill_attention(some, none, none, cumulative([5]), 0.1,
                                       cu_seqlens_k=cumulative([0])) == 0).all())
    x = np.random.default_rng(0).standard_normal((9, 2, 64)).astype(np.float16)
    got = ops.prefill_attention(x, x, x, np.array([0, 9], np.int32), 0.1)
    assert isinstance(got, np.ndarray)
    t = torch.from_numpy(x).cuda()
    np.testing.assert_array_equal(got, ops.prefill_attention(t, t, t, cumulative([9]), 0.1).cpu().numpy())


def test_refusals(cuda):
    from pagedkv_fusion import ops
    q = torch.ones(6, 4, 64, device="cuda", dtype=torch.float16)
    cu = cumulative([6])
    for args, kw, msg in [
        ((q.float(), q.float(), q.float(), cu, 0.1), {}, "float16"),
        ((q, q.bfloat16(), q, cu, 0.1), {}, "q's type"),
        ((q, q[..., :32], q[..., :32], cu, 0.1), {}, "q's type"),
        ((q, q, q[:, :2], cu, 0.1), {}, "q's type"),
        ((q, q[:, :3], q[:, :3], cu, 0.1), {}, "GQA"),
        ((q, q, q, cu.long(), 0.1), {}, "int32"),
        ((q, q, q, cu, 0.1), {"cu_seqlens_k": cumulative([3, 3])}, "cu_seqlens"),
        ((q, q, q, cu, 0.0), {}, "sm_scale"), ((q, q, q, cu, -1.0), {}, "sm_scale"),
        ((q, q, q, cu, float("nan")), {}, "sm_scale"),
        ((q[..., :12], q[..., :12], q[..., :12], cu, 0.1), {}, "head_dim"),
        ((q.clone().requires_grad_(), q, q, cu, 0.1), {}, "backward"),
    ]:
        with pytest.raises(RuntimeError, match=msg):
            ops.prefill_attention(*args, **kw)
    big = torch.ones(2, 1, 136, device="cuda", dtype=torch.float16)
    with pytest.raises(RuntimeError, match="head_dim"):
        ops.prefill_attention(big, big, big, cumulative([2]), 0.1)
