"""evict_tokens against the rule in NumPy: what stays is exact, the weights move bit for bit, the
scales are maxima, and codes are those of fp32 arithmetic, which in 64 bits differ from rounding
to nearest only where the product is within 2^-23 of itself of a half.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def problem(seed, lens, kv_heads, dim, bs, wide=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = [-(-max(n, 0) // bs) for n in lens]
    nb = sum(pages) + 3
    perm = torch.randperm(nb, generator=g, device="cuda").to(torch.int32)
    tables = torch.full((len(lens), max(pages, default=0) + wide), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(pages):
        tables[i, :n] = perm[at:at + n]
        at += n
    return dict(
        kv_cache_int8=torch.randint(-127, 128, (2, nb, bs, kv_heads, dim), generator=g, device="cuda",
                                    dtype=torch.int8),
        scale_cache=torch.exp(torch.randn(2, nb, kv_heads, generator=g, device="cuda")) / 60,
        weights=torch.rand(nb, bs, generator=g, device="cuda"), block_tables=tables,
        seq_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))


def order_key(w):
    """float32 weights as integers that sort alike, -0 with +0, NaN last."""
    u = np.where(w == 0, np.float32(0), w).view(np.uint32)
    key = np.where(u >> 31, ~u, u | 0x80000000)
    return np.where(np.isnan(w), 0xFFFFFFFF, key).astype(np.int64)


def expected(p, keep, sinks, recent):
    cache, scales, weights = (p[k].cpu().numpy().copy() for k in ("kv_cache_int8", "scale_cache", "weights"))
    tables, lens = p["block_tables"].cpu().numpy(), p["seq_lens"].cpu().numpy()
    bs = weights.shape[1]
    new_lens, kept = [], np.full((len(lens), keep), -1, np.int32)
    exact = cache.astype(np.float64)
    for i, n in enumerate(lens):
        n = max(int(n), 0)
        if n <= keep:
            new_lens.append(n)
            kept[i, :n] = np.arange(n)
            continue
        pages = tables[i, :-(-n // bs)]
        w = weights[pages].reshape(-1)[:n].copy()
        middle = np.argsort(-order_key(w[sinks:n - recent]), kind="stable")[:keep - sinks - recent]
        stay = np.concatenate([np.arange(sinks), np.sort(middle) + sinks, np.arange(n - recent, n)])
        new_lens.append(keep)
        kept[i] = stay
        old_codes = cache[:, pages].reshape(2, -1, *cache.shape[3:])[:, stay]
        old = scales[:, pages[stay // bs]]
        for j in range(-(-keep // bs)):
            part = slice(j * bs, min((j + 1) * bs, keep))
            size = part.stop - part.start
            new = old[:, part].max(1)
            ratio = old[:, part] / new[:, None]
            moved = np.rint(old_codes[:, part].astype(np.float32) * ratio[..., None])
            shrinks = (old[:, part] < new[:, None])[..., None]
            cache[:, pages[j], :size] = np.where(shrinks, moved, old_codes[:, part]).astype(np.int8)
            exact[:, pages[j], :size] = old_codes[:, part].astype(np.float64) * np.where(
                shrinks, (old[:, part].astype(np.float64) / new[:, None])[..., None], 1.0)
            scales[:, pages[j]] = new
        flat = weights[pages].reshape(-1)
        flat[:n] = 0
        flat[:keep] = w[stay]
        weights[pages] = flat.reshape(-1, bs)
    return cache, scales, weights, np.array(new_lens, np.int32), kept, exact


def run(p, keep, sinks=0, recent=0, error=0):
    from pagedkv_fusion import _C, ops
    got = {k: v.clone() for k, v in p.items()}
    lens, kept = ops.evict_tokens(**got, keep=keep, sinks=sinks, recent=recent)
    assert _C.read_device_error() == error
    return got, lens, kept


def check(p, keep, sinks=0, recent=0):
    got, lens, kept = run(p, keep, sinks, recent)
    cache, scales, weights, new_lens, stay, exact = expected(p, keep, sinks, recent)
    assert lens.dtype == torch.int32 and kept.dtype == torch.int32
    assert np.array_equal(lens.cpu().numpy(), new_lens) and np.array_equal(kept.cpu().numpy(), stay)
    assert np.array_equal(got["scale_cache"].cpu().numpy(), scales)
    assert np.array_equal(got["weights"].cpu().numpy(), weights, equal_nan=True)
    codes = got["kv_cache_int8"].cpu().numpy()
    assert np.array_equal(codes, cache)
    assert (np.abs(codes - exact) <= 0.5 + 2.0 ** -23 * 127).all()
    for k in ("block_tables", "seq_lens"):
        assert torch.equal(got[k], p[k])
    return got


@pytest.mark.parametrize("lens,keep,sinks,recent,kv_heads,dim,bs", [
    ([1], 1, 0, 0, 1, 32, 16), ([2], 1, 0, 0, 1, 64, 16), ([2], 1, 1, 0, 2, 64, 16), ([2], 1, 0, 1, 2, 64, 16),
    ([300, 100, 251], 128, 4, 32, 8, 64, 16), ([5, 0, 17, 16], 16, 3, 3, 2, 128, 16),
    ([1000, 999], 999, 10, 10, 8, 128, 16), ([777], 40, 40, 0, 4, 128, 32), ([777], 40, 0, 40, 4, 128, 32),
    ([777], 40, 20, 20, 4, 96, 32), ([500] * 5, 77, 1, 0, 3, 128, 5), ([200, 300], 150, 2, 9, 2, 80, 64),
    ([129], 64, 0, 1, 1, 256, 64), ([300], 111, 2, 2, 2, 100, 64), ([300, 40], 111, 2, 2, 2, 33, 16),
    ([90], 33, 0, 0, 2, 255, 64), ([2000] * 70, 700, 4, 100, 2, 32, 16), ([5000], 1500, 16, 64, 8, 128, 16),
    ([60], 30, 1, 2, 40, 128, 1), ([9000, 100, 4000], 3000, 4, 64, 1, 64, 48), ([40] * 200, 20, 2, 2, 2, 64, 8),
])
def test_matches_the_rule(cuda, lens, keep, sinks, recent, kv_heads, dim, bs):
    check(problem(1, lens, kv_heads, dim, bs, wide=len(lens) % 2), keep, sinks, recent)


def test_long_sequences(cuda):
    """More tokens than sort keys fit on chip, and few sequences of many."""
    check(problem(2, [70000, 300], 1, 32, 16), 20000, 4, 100)
    check(problem(3, [49152], 2, 64, 32), 49151, 0, 0)


def test_ties_zeros_and_not_finite_weights(cuda):
    p = problem(4, [400, 300, 350], 2, 64, 16)
    p["weights"].copy_(torch.round(p["weights"] * 4) / 4)  # few values: the earlier token stays
    check(p, 100, 3, 5)
    p["weights"].zero_()
    p["weights"][::2] = -0.0
    check(p, 100, 0, 0)
    p["weights"].uniform_(-1, 1)
    p["weights"][::3, ::2] = float("nan")
    p["weights"][1::3, 1::2] = float("inf")
    p["weights"][2::3, ::5] = -float("inf")
    for keep in (20, 100, 250):
        check(p, keep, 1, 1)


def test_scales_of_any_kind(cuda):
    """Zero, equal and infinite scales: codes move as they are where the old one is not smaller."""
    p = problem(5, [200, 150], 2, 64, 16)
    p["scale_cache"][:] = 0.01
    before = p["kv_cache_int8"].clone()
    got, lens, kept = run(p, 60, 2, 2)
    bs = 16
    for i in range(2):
        t = p["block_tables"][i].long()
        src, dst = kept[i].long(), torch.arange(60, device="cuda")
        moved = got["kv_cache_int8"][:, t[dst // bs], dst % bs]
        assert torch.equal(moved, before[:, t[src // bs], src % bs])
    p["scale_cache"][:, ::2] = 0.0
    check(p, 60, 2, 2)
    p["scale_cache"][0, ::3] = float("inf")
    got, _, _ = run(p, 60, 2, 2)
    assert bool((got["kv_cache_int8"] != -128).all())


def test_short_and_bad_sequences_stay(cuda):
    p = problem(6, [100, 60, 90], 2, 64, 16, wide=1)
    got, lens, kept = run(p, 100, 5, 5)
    for k in p:
        assert torch.equal(got[k], p[k])
    assert lens.tolist() == [100, 60, 90] and kept[1, 59:62].tolist() == [59, -1, -1]
    # a page outside the cache: that sequence stays, the others are cut
    whole, _, _ = run(p, 50, 5, 5)
    for bad in (-1, p["weights"].shape[0], 2 ** 31 - 1):
        b = dict(p, block_tables=p["block_tables"].clone())
        b["block_tables"][0, 3] = bad
        got, lens, kept = run(b, 50, 5, 5, error=1)
        assert lens.tolist() == [100, 50, 50] and bool((kept[0] == -1).all())
        for i, same in ((0, p), (1, whole), (2, whole)):
            t = p["block_tables"][i]
            t = t[t >= 0].long()
            assert torch.equal(got["kv_cache_int8"][:, t], same["kv_cache_int8"][:, t])
            assert torch.equal(got["weights"][t], same["weights"][t])
    # lengths beyond the table are cut to it, negative ones hold nothing
    b = dict(p, block_tables=p["block_tables"].clamp(min=0)[:1].contiguous(), seq_lens=p["seq_lens"][:1] * 0 + 2 ** 31 - 1)
    b["block_tables"][0, -1] = p["weights"].shape[0] - 1
    _, lens, _ = run(b, 50, 5, 5, error=4)
    assert lens.tolist() == [50]
    got, lens, kept = run(dict(p, seq_lens=p["seq_lens"] * 0 - 9), 50, 5, 5)
    assert lens.tolist() == [0, 0, 0] and bool((kept == -1).all())
    none = {k: (v[:0] if k in ("block_tables", "seq_lens") else v) for k, v in p.items()}
    _, lens, kept = run(none, 50)
    assert lens.shape == (0,) and kept.shape == (0, 50)
    _, lens, _ = run(dict(p, block_tables=p["block_tables"][:, :0], seq_lens=p["seq_lens"] * 0), 50)
    assert lens.tolist() == [0, 0, 0]


def test_again_and_again(cuda):
    """Cut, grown by new tokens and cut again: the rule holds on what the last cut left."""
    p = problem(7, [300, 280], 2, 128, 16)
    for n in (120, 100, 64):
        p = dict(check(p, n, 4, 16), seq_lens=torch.tensor([n + 40, n + 9], dtype=torch.int32, device="cuda"))
        p["weights"].add_(torch.rand_like(p["weights"]))


def test_large_cache_offsets(cuda):
    p = problem(8, [300], 8, 128, 16)
    want, lens, kept = run(p, 100, 4, 4)
    nb = (9 << 29) // (16 * 8 * 128)
    far = torch.linspace(0, nb - 1, p["weights"].shape[0], device="cuda").long()
    big = dict(p, kv_cache_int8=torch.empty(2, nb, 16, 8, 128, dtype=torch.int8, device="cuda"),
               scale_cache=torch.zeros(2, nb, 8, device="cuda"), weights=torch.zeros(nb, 16, device="cuda"))
    for k in ("kv_cache_int8", "scale_cache"):
        big[k][:, far] = p[k]
    big["weights"][far] = p["weights"]
    big["block_tables"] = far[p["block_tables"].long()].to(torch.int32)
    from pagedkv_fusion import ops
    lens2, kept2 = ops.evict_tokens(**big, keep=100, sinks=4, recent=4)
    assert torch.equal(kept, kept2) and torch.equal(lens, lens2)
    assert torch.equal(big["kv_cache_int8"][:, far], want["kv_cache_int8"])
    assert torch.equal(big["scale_cache"][:, far], want["scale_cache"])
    assert torch.equal(big["weights"][far], want["weights"])


def test_graph_and_integer_types(cuda):
    from pagedkv_fusion import ops
    p = problem(9, [400, 90, 1000], 8, 64, 16)
    want, lens, kept = run(p, 80, 4, 8)
    got = {k: v.clone() for k, v in p.items()}
    warm = {k: v.clone() for k, v in p.items()}
    ops.evict_tokens(**dict(warm, seq_lens=p["seq_lens"].long(),
                            block_tables=p["block_tables"].T.contiguous().T), keep=80, sinks=4, recent=8)
    for k in ("kv_cache_int8", "scale_cache", "weights"):
        assert torch.equal(warm[k], want[k])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.evict_tokens(**got, keep=80, sinks=4, recent=8)
    for _ in range(2):
        for k, v in p.items():
            got[k].copy_(v)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], lens) and torch.equal(out[1], kept)
        for k in ("kv_cache_int8", "scale_cache", "weights"):
            assert torch.equal(got[k], want[k])


def test_refusals(cuda):
    from pagedkv_fusion import ops
    p = problem(10, [50], 2, 64, 16)
    for change, message in [
            (dict(keep=0), "keep"), (dict(keep=5, sinks=3, recent=3), "keep"), (dict(keep=5, sinks=-1), "keep"),
            (dict(kv_cache_int8=p["kv_cache_int8"][0]), "kv_cache_int8"),
            (dict(kv_cache_int8=p["kv_cache_int8"].float()), "kv_cache_int8"),
            (dict(kv_cache_int8=p["kv_cache_int8"][..., ::2]), "contiguous"),
            (dict(scale_cache=p["scale_cache"].double()), "scale_cache"),
            (dict(scale_cache=p["scale_cache"][:1]), "scale_cache"), (dict(weights=p["weights"][:-1]), "weights"),
            (dict(weights=p["weights"].half()), "weights"), (dict(block_tables=p["block_tables"].long()), "block_tables"),
            (dict(seq_lens=p["seq_lens"].float()), "seq_lens"), (dict(weights=p["weights"].cpu()), "CUDA")]:
        with pytest.raises(RuntimeError, match=message):
            ops.evict_tokens(**dict(dict(p, keep=10), **change))
