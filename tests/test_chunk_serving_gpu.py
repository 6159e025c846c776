"""Chunked prompts, drafted tokens, gathered attention weights and evicted tokens together, as
a server uses them on one INT8 cache: each step is held to the definition on what the cache holds.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from test_chunk_gpu import compare, reference
from test_evict_tokens_gpu import expected as cut
from test_weights_gpu import expected as gathered

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv_heads,dtype", [(32, 8, torch.bfloat16), (6, 2, torch.float16)])
def test_prompt_in_chunks_then_evictions_between_decode_steps(cuda, heads, kv_heads, dtype):
    from pagedkv_fusion import ops
    from pagedkv_fusion.backend import PagedKVFusionBackend, PagedKVFusionMetadata
    g = torch.Generator(device="cuda").manual_seed(heads)
    S, bs, D, width = 3, 16, 128, 70
    be = PagedKVFusionBackend(fallback_backend=None)
    scale = 1.0 / math.sqrt(D)
    nb = S * width + 2
    tables = torch.randperm(nb, generator=g, device="cuda")[:S * width].view(S, width).to(torch.int32)
    cache = torch.zeros(2, nb, bs, kv_heads, D, dtype=torch.int8, device="cuda")
    scales = torch.zeros(2, nb, kv_heads, device="cuda")
    weights = torch.zeros(nb, bs, device="cuda")
    meta = PagedKVFusionMetadata(tables, torch.zeros(S, dtype=torch.int32, device="cuda"), scales[0], scales[1])

    def step(q_lens):
        """Appends q_lens new tokens, attends, gathers their weights; every result is checked."""
        nonlocal meta
        T = sum(q_lens)
        q, k, v = (torch.randn(T, h, D, generator=g, device="cuda").to(dtype) for h in (heads, kv_heads, kv_heads))
        old = meta.seq_lens.tolist()
        pos = torch.cat([torch.arange(a, a + n) for a, n in zip(old, q_lens)]).cuda()
        seq = torch.repeat_interleave(torch.arange(S), torch.tensor(q_lens)).cuda()
        slots = tables[seq, pos // bs].long() * bs + pos % bs
        be.append_to_cache(k, v, cache, scales, slots, bs)
        weights.view(-1)[slots] = 0.0  # a new token's, whoever had its place
        meta = PagedKVFusionMetadata(tables, meta.seq_lens + torch.tensor(q_lens, dtype=torch.int32, device="cuda"),
                                     scales[0], scales[1])
        cu = torch.tensor([0] + q_lens).cumsum(0).to(torch.int32).cuda()
        p = dict(q=q, k_cache_q=cache[0], k_scale=scales[0], v_cache_q=cache[1], v_scale=scales[1],
                 block_tables=tables, seq_lens=meta.seq_lens, cu_seqlens=cu, sm_scale=scale)
        out, lse = be.chunk_forward(q, cache, scales, meta, cu, scale, return_lse=True)
        compare(p, out, lse, reference(p))
        start = weights.clone()
        be.accumulate_weights(weights, q, cache, scales, meta, cu, scale, lse=lse)
        want, tol = gathered(p, start)
        assert bool(((weights.double() - want).abs() <= tol).all())
        if max(q_lens) == 1:  # and as the decode kernels answer it
            plain = be.decode_forward(q.float(), cache, scales, meta, scale)
            rows = torch.tensor([n > 0 for n in q_lens]).cuda()[seq]
            torch.testing.assert_close(out[rows].float(), plain[seq][rows], rtol=2 * torch.finfo(dtype).eps,
                                       atol=2e-3)
        assert cuda.read_device_error() == 0

    for q_lens in ([512, 300, 1], [400, 9, 512], [1, 1, 1], [4, 1, 6]):  # chunks, a step, drafted tokens
        step(q_lens)
    for keep in (256, 256, 100):
        before = dict(kv_cache_int8=cache.clone(), scale_cache=scales.clone(), weights=weights.clone(),
                      block_tables=tables, seq_lens=meta.seq_lens)
        want = cut(before, keep, 4, 64)
        meta = be.evict_tokens(cache, scales, weights, meta, keep, sinks=4, recent=64)
        for got, plain in zip((cache, scales, weights, meta.seq_lens), want):
            assert np.array_equal(got.cpu().numpy(), plain)
        for q_lens in ([1, 1, 1], [3, 1, 2], [33, 1, 8], [1, 1, 1]):
            step(q_lens)
    # the gathered weights rank whole pages too
    valid = torch.zeros(nb, bs, dtype=torch.bool, device="cuda")
    for i, n in enumerate(meta.seq_lens.tolist()):
        at = torch.arange(n, device="cuda")
        valid[tables[i, at // bs].long(), at % bs] = True
    used = valid.any(1)
    zero = torch.zeros(nb, device="cuda")
    scores = ops.eviction_scores(zero, zero, weights, valid, w_recency=0.0, w_frequency=0.0, w_attention=1.0)
    mean = (weights.double() * valid).sum(1)[used] / valid.sum(1)[used]
    torch.testing.assert_close(scores[used].double(), mean, rtol=1e-6, atol=0.0)


def test_decode_loop_as_one_graph(cuda):
    """Append, attend, gather and cut on buffers that never move: a captured step and the eager
    one leave the same cache."""
    from pagedkv_fusion import ops
    g = torch.Generator(device="cuda").manual_seed(5)
    S, bs, D, H, Hkv, width, keep = 4, 16, 64, 8, 2, 9, 96
    nb = S * width
    tables = torch.randperm(nb, generator=g, device="cuda").view(S, width).to(torch.int32)
    cu = torch.arange(S + 1, dtype=torch.int32, device="cuda")
    new = [torch.empty(S, h, D, device="cuda", dtype=torch.bfloat16) for h in (H, Hkv, Hkv)]

    def fresh():
        return dict(cache=torch.zeros(2, nb, bs, Hkv, D, dtype=torch.int8, device="cuda"),
                    scales=torch.zeros(2, nb, Hkv, device="cuda"), weights=torch.zeros(nb, bs, device="cuda"),
                    lens=torch.zeros(S, dtype=torch.int32, device="cuda"))

    def step(b):
        q, k, v = new
        slots = tables.gather(1, (b["lens"] // bs).long()[:, None])[:, 0].long() * bs + b["lens"] % bs
        ops.append_kv(k, v, b["cache"], b["scales"], slots, bs)
        b["lens"] += 1
        b["weights"].view(-1).index_fill_(0, slots, 0.0)
        args = (tables, b["lens"], cu, 0.125)
        out, lse = ops.chunk_attention(q, b["cache"][0], b["scales"][0], b["cache"][1], b["scales"][1], *args,
                                       return_lse=True)
        ops.accumulate_attention(b["weights"], q, b["cache"][0], b["scales"][0], *args, lse=lse)
        return out

    def shorten(b):
        lens, _ = ops.evict_tokens(b["cache"], b["scales"], b["weights"], tables, b["lens"], keep, 4, 16)
        b["lens"].copy_(lens)

    eager, replayed, warm = fresh(), fresh(), fresh()
    for x in new:
        x.normal_(generator=g)
    step(warm), shorten(warm)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    with torch.cuda.graph(graphs[0]):
        out = step(replayed)
    with torch.cuda.graph(graphs[1]):
        shorten(replayed)
    for k, v in fresh().items():
        replayed[k].copy_(v)
    for t in range(200):
        for x in new:
            x.normal_(generator=g)
        graphs[0].replay()
        assert torch.equal(step(eager), out), t
        if t % 40 == 39:
            shorten(eager)
            graphs[1].replay()
            for k in eager:
                assert torch.equal(eager[k], replayed[k]), (t, k)
    assert eager["lens"].max() <= keep + 40 and cuda.read_device_error() == 0
