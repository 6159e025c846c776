"""chunk_attention against softmax attention in 64 bits over the dequantized cache.

Tolerance, per output, with p the row's probabilities, A = sum_j p_j |v_j|, n keys, D
channels, steps 2^-23 (two half steps of fp32, since tensor cores cut sums):

* a score is a sum of up to 2 D products (hi and lo of fp32 queries) whose codes may come
  128 too large, taken off by one more sum: off by at most
  t = (2 D + 8) 2^-23 S, S = |scale| k_scale sum_d |q_d| (|code_d| + 256), largest over the
  row's keys, which with the exponential's and its argument's own 2^-19 is the relative
  error of every p;
* numerator and denominator are sums of n terms: 2 n 2^-23;
* p times its V scale is one fp16 number for 16-bit queries (2^-11), two for fp32 (2^-20);
  below the smallest step of fp16 it is off by half of that, which is 2^-30 of the largest p
  and the largest V scale;
* the result is rounded to its type (2^-11 fp16, 2^-8 bf16, 2^-24 fp32), or, below the
  type's smallest normal number, where the step no longer shrinks, by half of that step,
  r_sub: fp16's is 2^-24 below 2^-14, so 2^-25.

|got - want| <= A (2 t + 2^-18 + 2 n 2^-23 + r_p) + 2^-30 n max(p) max|v| + r_out |want| + r_sub

The log denominator is off by t + 2^-19 + n 2^-23 and the steps of its own 2^-22 |lse|.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def problem(seed, q_lens, lens, heads, kv_heads, dim, bs, dtype="bf16", wide=0, spread=0.5):
    """New tokens q_lens of sequences of lens cached tokens, on shuffled pages."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = [-(-n // bs) for n in lens]
    nb = sum(pages) + 2
    perm = torch.randperm(nb, generator=g, device="cuda").to(torch.int32)
    width = max(pages, default=0) + wide
    tables = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(pages):
        tables[i, :n] = perm[at:at + n]
        at += n
    shape = (nb, bs, kv_heads, dim)
    codes = [torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8) for _ in "kv"]
    scales = [torch.exp(spread * torch.randn(nb, kv_heads, generator=g, device="cuda")) / 60
              for _ in "kv"]
    q = torch.randn(sum(q_lens), heads, dim, generator=g, device="cuda").to(TYPES[dtype])
    cu = torch.tensor([0] + list(q_lens), device="cuda").cumsum(0).to(torch.int32)
    return dict(q=q, k_cache_q=codes[0], k_scale=scales[0], v_cache_q=codes[1], v_scale=scales[1],
                block_tables=tables, seq_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                cu_seqlens=cu, sm_scale=1.0 / math.sqrt(dim))


def reference(p, lost=None):
    """(want, tolerance, lse, its tolerance, and of each (sequence, head) its rows, number of keys,
    probabilities and scores' errors); `lost` is a (sequence, page) that is not attended."""
    q = p["q"].double()
    bs, kv = p["k_cache_q"].shape[1:3]
    group, D = q.shape[1] // kv, q.shape[2]
    want, tol = torch.zeros_like(q), torch.zeros_like(q)
    lse = q.new_full(q.shape[:2], -math.inf)
    lse_tol, parts = torch.zeros_like(lse), []
    half = torch.finfo(p["q"].dtype).eps / 2
    sub = torch.finfo(p["q"].dtype).tiny * half
    r_p = 2.0 ** -20 if p["q"].dtype == torch.float32 else 2.0 ** -11
    cu = p["cu_seqlens"].tolist()
    for i, n in enumerate(p["seq_lens"].tolist()):
        a, b = cu[i], cu[i + 1]
        if b == a or n == 0:
            continue
        pages = p["block_tables"][i, :-(-n // bs)].long()
        seen = torch.ones(b - a, n, dtype=torch.bool, device=q.device).tril(n - (b - a))
        if lost is not None and lost[0] == i:
            seen[:, lost[1] * bs:(lost[1] + 1) * bs] = False

        def tokens(cache, scale, h):
            x = cache[pages, :, h].double()
            return x.flatten(0, 1)[:n], scale[pages, h].double().repeat_interleave(bs)[:n, None]

        for h in range(kv):
            kc, ks = tokens(p["k_cache_q"], p["k_scale"], h)
            vc, vs = tokens(p["v_cache_q"], p["v_scale"], h)
            v = vc * vs
            for j in range(h * group, (h + 1) * group):
                x = q[a:b, j]
                s = torch.where(seen, x @ (kc * ks).T * p["sm_scale"], -math.inf)
                S = (x.abs() @ ((kc.abs() + 256) * ks.abs()).T * abs(p["sm_scale"]))
                t = (2 * D + 8) * 2.0 ** -23 * torch.where(seen, S, 0.0).amax(1)
                lse[a:b, j] = torch.logsumexp(s, 1)
                w = torch.softmax(s, 1).nan_to_num(0.0)
                want[a:b, j] = w @ v
                tol[a:b, j] = (w @ v.abs()) * (2 * t + 2.0 ** -18 + 2 * n * 2.0 ** -23 + r_p)[:, None] + \
                    2.0 ** -30 * n * (w.amax(1) * v.abs().max())[:, None] + half * want[a:b, j].abs() + sub
                lse_tol[a:b, j] = t + 2.0 ** -19 + n * 2.0 ** -23 + 2.0 ** -22 * lse[a:b, j].abs().nan_to_num(0, 0, 0)
                parts.append((i, j, slice(a, b), n, w, t))
    return want, tol, lse, lse_tol, parts


def compare(p, out, lse, ref=None):
    want, tol, want_lse, lse_tol, _ = ref or reference(p)
    assert out.dtype == p["q"].dtype and out.shape == p["q"].shape and out.is_contiguous()
    bad = ~((out.double() - want).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float((out - want).abs().max()), bad.nonzero()[:5].tolist())
    none = want_lse == -math.inf
    assert bool((lse[none] == -math.inf).all()) and bool((out[none] == 0).all())
    bad = ~((lse.double() - want_lse).abs() <= lse_tol) & ~none
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:5].tolist())


def check(p, error=0):
    from pagedkv_fusion import _C, ops
    out, lse = ops.chunk_attention(**p, return_lse=True)
    assert _C.read_device_error() == error
    compare(p, out, lse)
    again = ops.chunk_attention(**p)
    assert torch.equal(out, again)  # the same bits every time, and with or without lse
    return out, lse


SHAPES = [
    # one token, one sequence
    ([1], [1], 1, 1, 32, 16), ([1], [700], 8, 8, 64, 16), ([1], [129], 4, 2, 128, 5),
    # decode of several, lengths of zero and of whole steps among them
    ([1] * 7, [0, 1, 15, 16, 17, 300, 64], 32, 8, 128, 16),
    ([1] * 40, [3 + 37 * i for i in range(40)], 16, 2, 96, 8),
    # a few tokens: several blocks of 8 rows
    ([3, 1, 8, 2], [50, 1, 1000, 2], 12, 4, 128, 32), ([5, 7], [400, 7], 14, 2, 64, 64),
    # chunks: whole units, units that end early, sequences of no new token
    ([300], [300], 8, 2, 128, 16), ([70, 0, 33, 1], [900, 40, 33, 600], 32, 8, 128, 16),
    ([129, 64], [500, 64], 8, 8, 64, 16), ([40], [3000], 40, 40, 128, 16),
    ([200], [2100], 6, 2, 96, 48), ([64], [5000], 1, 1, 32, 16),
    # more new tokens than cached ones: the first see nothing
    ([50, 3], [20, 1], 8, 2, 128, 16), ([10], [0], 8, 2, 128, 16),
    # wide groups, page sizes and head dims that only the warps take
    ([2, 1], [100, 333], 66, 2, 64, 16), ([9], [77], 33, 1, 128, 16), ([60], [300], 4, 2, 160, 16),
    ([1, 40], [500, 60], 8, 1, 256, 16), ([33, 1, 1], [200, 9, 70], 8, 2, 128, 1), ([100], [333], 8, 4, 128, 24),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("q_lens,lens,heads,kv_heads,dim,bs", SHAPES)
def test_matches_reference(cuda, dtype, q_lens, lens, heads, kv_heads, dim, bs):
    check(problem(1, q_lens, lens, heads, kv_heads, dim, bs, dtype, wide=len(lens) % 3))


@pytest.mark.parametrize("dtype,dim", [("f32", 64), ("f32", 128), ("f16", 64), ("bf16", 128)])
def test_sums_over_many_tiles(cuda, dtype, dim):
    """O is started anew every 5 (fp32) or 128 tiles of 128 keys; V of one sign would show what
    is cut or lost."""
    p = problem(2, [40, 2], [17100, 4000], 2, 1, dim, 32, dtype, spread=0.1)
    p["v_cache_q"].abs_()
    check(p)


def test_many_sequences(cuda):
    r = np.random.default_rng(3)
    q_lens = r.integers(0, 4, 600).tolist()
    lens = [int(n + r.integers(0, 60)) for n in q_lens]
    check(problem(3, q_lens, lens, 4, 2, 64, 16, "f16"))
    q_lens = r.integers(0, 60, 300).tolist()
    check(problem(4, q_lens, [n + 20 for n in q_lens], 8, 2, 64, 16, "bf16"))


def test_agrees_with_decode(cuda):
    from pagedkv_fusion import ops
    p = problem(5, [1] * 9, [5, 700, 33, 64, 1, 2000, 100, 16, 17], 32, 8, 128, 16, "f32")
    out = ops.chunk_attention(**p)
    args = {k: v for k, v in p.items() if k != "cu_seqlens"}
    torch.testing.assert_close(out, ops.quant_paged_attention(**args), rtol=2e-5, atol=2e-5)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_score_ranges_and_signs(cuda, dtype):
    """Rows from 2^-40 to 2^20 of one another, scores up to hundreds, negative scales, a scale
    of zero, rising and falling maxima."""
    for q_lens, lens in (([1, 2], [900, 333]), ([90], [1500]), ([200], [1500])):
        p = problem(6, q_lens, lens, 8, 2, 128, 16, dtype)
        rows = p["q"].shape[0] * 8
        scale = torch.tensor([2.0 ** -40, 2.0 ** -12, 1.0, 8.0, 0.0, 2.0 ** -5, 3.0, 2.0 ** -20])
        p["q"] *= scale.repeat(-(-rows // 8))[:rows].view(-1, 8, 1).cuda()
        p["k_scale"][::3] *= -1
        p["k_scale"][::7] = 0.0
        p["v_scale"][::5] *= -1
        p["v_scale"][1::4] *= 2.0 ** -30
        check(p)
        ramp = torch.linspace(0.01, 4.0, lens[0], device="cuda")
        for order in (ramp, ramp.flip(0)):
            pages = p["block_tables"][0, :-(-lens[0] // 16)].long()
            p["k_scale"][pages] = order[::16][:, None] / 40
            check(p)


def test_values_behind_a_row_do_not_reach_it(cuda):
    """Scales that are not finite on pages that only later tokens see, and stale ones."""
    from pagedkv_fusion import ops
    for q_lens, lens, heads in (([6], [40], 8), ([6], [36], 8), ([100], [230], 8), ([100], [230], 1),
                                ([300], [500], 8), ([330], [509], 8), ([600], [900], 1), ([50], [1500], 8)):
        p = problem(7, q_lens, lens, heads, 1, 128, 16, "f16", wide=2)
        want, want_lse = ops.chunk_attention(**p, return_lse=True)
        last = (lens[0] - 1) // 16  # the last page's tokens: seen from their own places on
        first_row = max(last * 16 - (lens[0] - q_lens[0]), 0)
        for name in ("k_scale", "v_scale"):
            for bad in (math.nan, math.inf):
                broken = dict(p, **{name: p[name].clone()})
                broken[name][p["block_tables"][0, last].long()] = bad
                out, lse = ops.chunk_attention(**broken, return_lse=True)
                assert torch.equal(out[:first_row], want[:first_row])
                assert torch.equal(lse[:first_row], want_lse[:first_row])
                assert not bool(torch.isfinite(out[first_row:].float()).any(-1).all())
                if name == "v_scale":
                    assert torch.equal(lse, want_lse)
        # pages that are in no table, and table entries behind the length
        q = dict(p, block_tables=p["block_tables"].clone())
        q["block_tables"][:, last + 1:] = 123456789
        other = torch.ones(p["k_scale"].shape[0], dtype=torch.bool)
        other[p["block_tables"][0, :last + 1].cpu().long()] = False
        for name in ("k_scale", "v_scale"):
            q[name] = p[name].clone()
            q[name][other.cuda()] = math.nan
        out, lse = ops.chunk_attention(**q, return_lse=True)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
    assert cuda.read_device_error() == 0


def test_rows_do_not_touch_each_other(cuda):
    from pagedkv_fusion import ops
    for q_lens, lens in (([1, 1, 3], [100, 30, 50]), ([80], [700]), ([300], [700]), ([30], [6000])):
        p = problem(8, q_lens, lens, 8, 2, 128, 16, "bf16")
        want = ops.chunk_attention(**p)
        for bad in (math.nan, math.inf, 3e38):
            broken = dict(p, q=p["q"].clone())
            broken["q"][1, 2] = bad
            out = ops.chunk_attention(**broken)
            assert not bool(torch.isfinite(out[1, 2].float()).all()) or bad == 3e38
            out[1, 2] = want[1, 2]
            assert torch.equal(out, want)


def test_rows_outside_sequences_become_zero(cuda):
    from pagedkv_fusion import ops
    for q_lens, lens in (([1] * 5, [9] * 5), ([70, 40], [200, 40]), ([300, 40, 1], [700, 40, 90])):
        p = problem(9, q_lens, lens, 8, 2, 128, 16, "f16")
        want, want_lse = ops.chunk_attention(**p, return_lse=True)
        pad = torch.full((3, 8, 128), math.nan, dtype=torch.float16, device="cuda")
        out, lse = ops.chunk_attention(**dict(p, q=torch.cat([pad, p["q"], pad]),
                                              cu_seqlens=p["cu_seqlens"] + 3), return_lse=True)
        assert torch.equal(out[3:-3], want) and torch.equal(lse[3:-3], want_lse)
        for part in (slice(0, 3), slice(-3, None)):
            assert bool((out[part] == 0).all()) and bool((lse[part] == -math.inf).all())
    # no sequence at all
    none = dict(p, block_tables=p["block_tables"][:0], seq_lens=p["seq_lens"][:0],
                cu_seqlens=p["cu_seqlens"][:1])
    out, lse = ops.chunk_attention(**none, return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    empty = dict(p, q=p["q"][:0], cu_seqlens=p["cu_seqlens"] * 0)
    assert ops.chunk_attention(**empty).shape == (0, 8, 128)
    assert cuda.read_device_error() == 0


def test_bad_pages_lengths_and_cu_seqlens(cuda):
    from pagedkv_fusion import ops
    for q_lens, lens, bs in (([1, 2], [100, 60], 16), ([1, 2], [100, 60], 5), ([90, 50], [300, 60], 16), ([300, 50], [700, 2000], 16)):
        p = problem(10, q_lens, lens, 8, 2, 128, bs, "f32")
        # a page outside the cache: its tokens are not attended
        for bad in (-1, p["k_scale"].shape[0], 2 ** 31 - 1):
            broken = dict(p, block_tables=p["block_tables"].clone())
            broken["block_tables"][0, 1] = bad
            out, lse = ops.chunk_attention(**broken, return_lse=True)
            assert cuda.read_device_error() == 1
            compare(p, out, lse, reference(p, lost=(0, 1)))
        # a length beyond the table
        long = dict(p, seq_lens=p["seq_lens"].clone())
        long["seq_lens"][0] = 2 ** 31 - 1
        cut = dict(p, seq_lens=p["seq_lens"].clone())
        cut["seq_lens"][0] = p["block_tables"].shape[1] * bs
        table = p["block_tables"].clamp(min=0)
        out = ops.chunk_attention(**dict(long, block_tables=table))
        assert cuda.read_device_error() == 4
        assert torch.equal(out, ops.chunk_attention(**dict(cut, block_tables=table)))
        # negative lengths hold nothing
        out = ops.chunk_attention(**dict(p, seq_lens=p["seq_lens"] * 0 - 7))
        assert bool((out == 0).all()) and cuda.read_device_error() == 0
        # cu_seqlens that fall, or pass the tensor, are cut
        T = p["q"].shape[0]
        for cu, same in (([0, 2 * T, 2 * T], [0, T, T]), ([-5, 1, T], [0, 1, T]), ([0, T, 1], [0, T, T])):
            cu, same = (torch.tensor(c, dtype=torch.int32, device="cuda") for c in (cu, same))
            out = ops.chunk_attention(**dict(p, cu_seqlens=cu))
            assert cuda.read_device_error() == 6
            assert torch.equal(out, ops.chunk_attention(**dict(p, cu_seqlens=same)))
    assert cuda.read_device_error() == 0


def test_strides_alignment_and_integer_types(cuda):
    """Views of one projection's output, odd addresses, tables and lengths of other layouts."""
    from pagedkv_fusion import ops
    for q_lens, lens, dtype in (([1, 3], [50, 70], "bf16"), ([60, 9], [300, 10], "f16"), ([40], [90], "f32"),
                                ([300, 9], [900, 10], "bf16"), ([300], [800], "f32")):
        p = problem(11, q_lens, lens, 8, 2, 64, 16, dtype)
        want = ops.chunk_attention(**p)
        T = p["q"].shape[0]
        wide = torch.randn(T, 12, 64, device="cuda").to(p["q"].dtype)
        wide[:, 2:10] = p["q"]
        views = [wide[:, 2:10], p["q"].transpose(0, 1).contiguous().transpose(0, 1),
                 p["q"].permute(2, 0, 1).contiguous().permute(1, 2, 0)]
        odd = torch.empty(p["q"].numel() + 1, dtype=p["q"].dtype, device="cuda")[1:]
        views.append(odd.copy_(p["q"].flatten()).view_as(p["q"]))
        for v in views:
            assert torch.equal(ops.chunk_attention(**dict(p, q=v)), want)
        more = dict(p, seq_lens=p["seq_lens"].long(),
                    block_tables=p["block_tables"].T.contiguous().T,
                    k_scale=p["k_scale"].T.contiguous().T,
                    cu_seqlens=torch.stack([p["cu_seqlens"]] * 2, 1)[:, 0])
        caches = torch.stack([p["k_cache_q"], p["v_cache_q"]])
        more.update(k_cache_q=caches[0], v_cache_q=caches[1])
        assert torch.equal(ops.chunk_attention(**more), want)
        shifted = torch.empty(p["k_cache_q"].numel() + 1, dtype=torch.int8, device="cuda")[1:]
        more["k_cache_q"] = shifted.copy_(p["k_cache_q"].flatten()).view_as(p["k_cache_q"])
        assert torch.equal(ops.chunk_attention(**more), want)


def test_strides_of_single_rows(cuda):
    """Dimensions of one have whatever stride their view left them: contiguous, but not to step by."""
    from pagedkv_fusion import ops
    for q_lens, lens, heads, kv_heads in (([1], [50], 8, 2), ([5], [70], 1, 1), ([1], [9], 1, 1)):
        p = problem(18, q_lens, lens, heads, kv_heads, 64, 16, "bf16")
        want = ops.chunk_attention(**p)
        q = p["q"].as_strided(p["q"].shape, (p["q"].stride(0) if len(p["q"]) > 1 else 7,
                                             p["q"].stride(1) if heads > 1 else 13, 1))
        assert torch.equal(q, p["q"]) and torch.equal(ops.chunk_attention(**dict(p, q=q)), want)
        weights = torch.zeros(p["k_cache_q"].shape[:2], device="cuda")
        same = weights.clone()
        args = {k: v for k, v in p.items() if not k.startswith("v_") and k != "q"}
        ops.accumulate_attention(weights, p["q"], **args)
        ops.accumulate_attention(same, q, **args)
        assert torch.equal(weights, same)


def test_large_cache_offsets(cuda):
    """Pages more than 2^32 bytes apart."""
    from pagedkv_fusion import ops
    for q_lens, lens, bs in (([1, 2], [100, 60], 16), ([90], [200], 16), ([300], [500], 16), ([2], [50], 8)):
        p = problem(12, q_lens, lens, 8, 8, 128, bs, "bf16")
        nb = (9 << 29) // (bs * 8 * 128)  # 4.8 GB
        far = torch.linspace(0, nb - 1, p["k_scale"].shape[0], device="cuda").long()
        big = dict(p)
        for name in ("k_cache_q", "v_cache_q"):
            big[name] = torch.empty(nb, bs, 8, 128, dtype=torch.int8, device="cuda")
            big[name][far] = p[name]
        for name in ("k_scale", "v_scale"):
            big[name] = torch.zeros(nb, 8, device="cuda")
            big[name][far] = p[name]
        big["block_tables"] = torch.where(p["block_tables"] >= 0, far[p["block_tables"].clamp(min=0).long()],
                                          -1).to(torch.int32)
        assert torch.equal(ops.chunk_attention(**big), ops.chunk_attention(**p))
        del big


def test_graph_follows_lengths_and_streams_do_not_mix(cuda):
    """A captured call follows its tensors; two graphs and an eager call on other streams share
    nothing."""
    from pagedkv_fusion import ops
    a = problem(13, [1] * 6, [700, 30, 1, 64, 200, 9], 32, 8, 128, 16, "bf16", wide=1)
    b = problem(14, [60, 3], [900, 40], 8, 2, 128, 16, "f16")
    c = problem(17, [300, 3, 90], [900, 40, 2000], 8, 2, 128, 16, "f32")
    problems, graphs, outs = [a, b, c], [], []
    for p in problems:
        ops.chunk_attention(**p)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.chunk_attention(**p, return_lse=True))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in problems]
    for lens in ([700, 30, 1, 64, 200, 9], [5, 704, 0, 1, 33, 64]):
        a["seq_lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        a["block_tables"].clamp_(min=0)
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                for _ in range(3):
                    g.replay()
        eager = [ops.chunk_attention(**p, return_lse=True) for p in problems]
        torch.cuda.synchronize()
        for p, got, plain in zip(problems, outs, eager):
            assert torch.equal(got[0], plain[0]) and torch.equal(got[1], plain[1])
            compare(p, *got)


def test_host_inputs_are_staged(cuda):
    from pagedkv_fusion import ops
    p = problem(15, [2, 1], [30, 9], 4, 2, 64, 16, "f32")
    want, lse = ops.chunk_attention(**p, return_lse=True)
    host = {k: v.cpu().numpy() if torch.is_tensor(v) else v for k, v in p.items()}
    got = ops.chunk_attention(**host, return_lse=True)
    assert np.array_equal(got[0], want.cpu().numpy()) and np.array_equal(got[1], lse.cpu().numpy())


def test_refusals(cuda):
    from pagedkv_fusion import ops
    p = problem(16, [2, 1], [30, 9], 4, 2, 64, 16, "f16")
    f = p["k_cache_q"]
    for change, message in [
            (dict(q=p["q"][0]), "q must be"), (dict(q=p["q"].double()), "q must be"),
            (dict(q=p["q"][:, :3]), "multiple of num_kv_heads"), (dict(q=p["q"][..., :32]), "head_dim"),
            (dict(k_cache_q=f.float()), "int8"), (dict(v_cache_q=f[:-1]), "shaped like"),
            (dict(v_cache_q=f.float()), "shaped like"), (dict(k_scale=p["k_scale"].double()), "scales"),
            (dict(v_scale=p["v_scale"][:, :1]), "scales"), (dict(block_tables=p["block_tables"].long()), "block_tables"),
            (dict(seq_lens=p["seq_lens"].float()), "seq_lens"), (dict(seq_lens=p["seq_lens"][:1]), "seq_lens"),
            (dict(cu_seqlens=p["cu_seqlens"].long()), "cu_seqlens"), (dict(cu_seqlens=p["cu_seqlens"][:2]), "cu_seqlens"),
            (dict(q=p["q"].clone().requires_grad_()), "no backward")]:
        with pytest.raises(RuntimeError, match=message):
            ops.chunk_attention(**dict(p, **change))
    odd = torch.zeros(3, 16, 2, 48, dtype=torch.int8, device="cuda")
    with pytest.raises(RuntimeError, match="head_dim % 32"):
        ops.chunk_attention(**dict(p, q=torch.zeros(3, 4, 48, device="cuda"), k_cache_q=odd, v_cache_q=odd))
    odd = torch.zeros(3, 65, 2, 64, dtype=torch.int8, device="cuda")
    with pytest.raises(RuntimeError, match="block_size"):
        ops.chunk_attention(**dict(p, k_cache_q=odd, v_cache_q=odd))
    with torch.no_grad():
        ops.chunk_attention(**dict(p, q=p["q"].clone().requires_grad_()))
