"""The prompt and shared-prefix operators together, as a server uses them:
a common prompt is projected, normed and rotated, attended and appended to the
INT8 cache once; then each sequence's new tokens are normed and rotated,
appended, and decoded over [shared prefix | own tokens], eagerly and as one
captured graph.

Each operator is held to the definition on its own inputs (tolerances in the
operators' own tests); the attention over the cache is compared with 64-bit
attention over the values that the cache holds.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from test_prefill_gpu import cumulative
from test_prefill_gpu import reference as prompt_reference
from test_prefix_gpu import reference as prefix_reference
from test_rotary_gpu import assert_rope_close, expected_qk, np_append

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv_heads,dtype,prompt", [(32, 8, torch.bfloat16, 333),
                                                         (6, 2, torch.float16, 1500)])
def test_prompt_then_decode_behind_a_shared_prefix(cuda, heads, kv_heads, dtype, prompt):
    from pagedkv_fusion import ops
    from pagedkv_fusion.backend import PagedKVFusionBackend, PagedKVFusionMetadata
    g = torch.Generator(device="cuda").manual_seed(heads)
    S, bs, D, width = 5, 16, 128, 3
    be = PagedKVFusionBackend(fallback_backend=None)
    scale = 1.0 / math.sqrt(D)
    table = ops.rotary_table(prompt + 64, D)
    qw, kw = (1 + 0.1 * torch.randn(2, D, generator=g, device="cuda")).to(dtype)

    def project(n):
        qkv = torch.randn(n, heads + 2 * kv_heads, D, generator=g, device="cuda").to(dtype)
        return qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]

    shared = -(-prompt // bs)
    nb = shared + S * width + 2
    perm = torch.randperm(nb, generator=g, device="cuda").to(torch.int32)
    prefix_table, tables = perm[:shared], perm[shared:shared + S * width].view(S, width).contiguous()
    cache = torch.zeros(2, nb, bs, kv_heads, D, dtype=torch.int8, device="cuda")
    scales = torch.zeros(2, nb, kv_heads, device="cuda")
    cache_h, scales_h = cache.cpu().numpy(), scales.cpu().numpy()

    # the prompt, once
    q, k, v = project(prompt)
    pos = torch.arange(prompt, device="cuda")
    q2, k2 = ops.qk_norm_rope(q, k, pos, table, qw, kw)
    assert_rope_close(q2, expected_qk(q, pos, table, qw, 1e-6, False), dtype)
    assert_rope_close(k2, expected_qk(k, pos, table, kw, 1e-6, False), dtype)
    out = be.prefill_forward(q2, k2, v, cumulative([prompt]), scale)
    want, _, tol = prompt_reference(q2, k2, v, [prompt], [prompt], scale, True)
    assert bool(((out.double() - want).abs() <= tol).all())
    slots = prefix_table[pos // bs].long() * bs + pos % bs
    be.append_to_cache(k2, v, cache, scales, slots, bs)
    np_append(k2.float().cpu().numpy(), v.float().cpu().numpy(), cache_h, scales_h,
              slots.cpu().numpy(), bs)
    np.testing.assert_array_equal(cache.cpu().numpy(), cache_h)

    # decode steps; the graph reads the same buffers
    tok = project(S)
    bufs = dict(q=tok[0].clone(), k=tok[1].clone(), v=tok[2].clone(),
                pos=torch.full((S,), prompt, device="cuda"),
                slots=torch.zeros(S, dtype=torch.int64, device="cuda"))
    lens = torch.zeros(S, dtype=torch.int32, device="cuda")
    plen = torch.tensor([prompt], dtype=torch.int32, device="cuda")
    meta = PagedKVFusionMetadata(tables, lens, scales[0], scales[1])

    def step():
        qs, _ = ops.qk_norm_rope(bufs["q"], None, bufs["pos"], table, qw)
        # without a norm on the keys, the append rotates them
        be.append_to_cache(bufs["k"], bufs["v"], cache, scales, bufs["slots"], bs,
                           positions=bufs["pos"], rotary=table)
        return be.shared_prefix_forward(qs.float(), cache, scales, meta, prefix_table, plen, scale)

    graph, replayed = None, None
    for t in range(20):
        for name, x in zip("qkv", project(S)):
            bufs[name].copy_(x)
        own = torch.arange(S, device="cuda") % 3 + t          # uneven own lengths
        bufs["pos"].copy_(prompt + own)
        bufs["slots"].copy_(tables[torch.arange(S, device="cuda"), own // bs].long() * bs + own % bs)
        lens.copy_(own + 1)
        if t == 0:  # tokens before the first one of a sequence: offsets 0 .. own - 1
            for i in range(S):
                for o in range(int(own[i])):
                    args = (bufs["k"][i:i + 1], bufs["v"][i:i + 1], cache, scales,
                            tables[i, :1].long() * bs + o, bs)
                    at = torch.tensor([prompt + o], device="cuda")
                    be.append_to_cache(*args, positions=at, rotary=table)
                    np_append(*(x.float().cpu().numpy() for x in args[:2]), cache_h, scales_h,
                              args[4].cpu().numpy(), bs, table[at].cpu().numpy())
        before = cache.clone(), scales.clone()
        out = step()
        if graph is None:
            graph = torch.cuda.CUDAGraph()
            cache.copy_(before[0]), scales.copy_(before[1])
            with torch.cuda.graph(graph):
                replayed = step()
        cache.copy_(before[0]), scales.copy_(before[1])
        graph.replay()
        assert torch.equal(replayed, out), t
        np_append(bufs["k"].float().cpu().numpy(), bufs["v"].float().cpu().numpy(), cache_h, scales_h,
                  bufs["slots"].cpu().numpy(), bs, table[bufs["pos"]].cpu().numpy())
        np.testing.assert_array_equal(cache.cpu().numpy(), cache_h)
        np.testing.assert_array_equal(scales.cpu().numpy().view(np.uint32), scales_h.view(np.uint32))
        qs, _ = ops.qk_norm_rope(bufs["q"], None, bufs["pos"], table, qw)
        want, tol = prefix_reference(dict(
            q=qs.float(), k_cache_q=cache[0], k_scale=scales[0], v_cache_q=cache[1],
            v_scale=scales[1], prefix_table=prefix_table, prefix_len=plen, block_tables=tables,
            seq_lens=lens, sm_scale=scale))
        assert bool(((out.double() - want).abs() <= tol).all()), t
    assert cuda.read_device_error() == 0


def test_chunked_prompt_equals_whole(cuda):
    """A prompt attended in chunks against its growing keys gives the rows of
    the whole prompt: each row sees the same keys, so only the roundings of the
    row maxima's order differ, within the operator's tolerance of either."""
    from pagedkv_fusion import ops
    g = torch.Generator(device="cuda").manual_seed(2)
    q = torch.randn(900, 8, 64, generator=g, device="cuda").half()
    k, v = torch.randn(2, 900, 2, 64, generator=g, device="cuda").half()
    whole = ops.prefill_attention(q, k, v, cumulative([900]), 0.125)
    _, _, tol = prompt_reference(q, k, v, [900], [900], 0.125, True)
    at = 0
    for n in (1, 255, 300, 344):
        part = ops.prefill_attention(q[at:at + n], k[:at + n], v[:at + n], cumulative([n]), 0.125,
                                     cu_seqlens_k=cumulative([at + n]))
        assert bool(((part.double() - whole[at:at + n].double()).abs() <= 2 * tol[at:at + n]).all())
        at += n


def test_two_streams_at_once(cuda):
    """The same operators from two streams, each with its own tensors, give what
    they give alone."""
    from pagedkv_fusion import ops
    jobs = []
    for seed in (1, 2):
        g = torch.Generator(device="cuda").manual_seed(seed)
        q = torch.randn(700, 8, 128, generator=g, device="cuda").bfloat16()
        k, v = torch.randn(2, 700, 2, 128, generator=g, device="cuda").bfloat16()
        table = ops.rotary_table(700, 128)
        slots = torch.randperm(48 * 16, generator=g, device="cuda")[:700]

        def job(q=q, k=k, v=v, table=table, slots=slots):
            pos = torch.arange(700, device="cuda")
            q2, k2 = ops.qk_norm_rope(q, k, pos, table)
            out = ops.prefill_attention(q2, k2, v, cumulative([300, 400]), 0.09)
            cache = torch.zeros(2, 48, 16, 2, 128, dtype=torch.int8, device="cuda")
            scales = torch.ones(2, 48, 2, device="cuda")
            ops.append_kv(k, v, cache, scales, slots, 16, pos, table)
            pages = torch.arange(40, dtype=torch.int32, device="cuda")
            dec = ops.shared_prefix_attention(
                q[:32].float(), cache[0], scales[0], cache[1], scales[1], pages,
                torch.tensor([640], device="cuda"), pages[:32, None].contiguous(),
                torch.full((32,), 9, dtype=torch.int32, device="cuda"), 0.09)
            return out, cache, scales, dec
        jobs.append(job)
    alone = [job() for job in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(3):
        for st, job in zip(streams, jobs):
            with torch.cuda.stream(st):
                got.append(job())
    torch.cuda.synchronize()
    for i, res in enumerate(got):
        for a, b in zip(res, alone[i % 2]):
            assert torch.equal(a, b)
    assert cuda.read_device_error() == 0
