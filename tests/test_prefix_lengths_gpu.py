"""shared_prefix_attention's lengths beyond its tables, tables without any
page among them: cut to the table and reported.
"""

from __future__ import annotations

import pytest
import torch

from test_prefix_gpu import problem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv_heads,dim,bs", [(8, 2, 128, 16), (6, 2, 96, 16), (4, 4, 64, 8)])
def test_lengths_beyond_tables_without_pages(cuda, heads, kv_heads, dim, bs):
    from pagedkv_fusion import ops
    p = problem(1, 100, [9, 0, 30], heads, kv_heads, dim, bs)
    none = dict(prefix_table=p["prefix_table"][:0], block_tables=p["block_tables"][:, :0])

    def call(**kw):
        return ops.shared_prefix_attention(**dict(p, **kw))

    zero = torch.zeros_like(p["seq_lens"])
    want = call(prefix_len=torch.zeros_like(p["prefix_len"]))
    assert cuda.read_device_error() == 0
    # a prefix without pages
    assert torch.equal(call(prefix_table=none["prefix_table"]), want)
    assert cuda.read_device_error() == 4
    for n in (0, -5):
        length = torch.full_like(p["prefix_len"], n)
        assert torch.equal(call(prefix_table=none["prefix_table"], prefix_len=length), want)
        assert cuda.read_device_error() == 0
    # own tokens without pages: any one of the sequences
    want = call(seq_lens=zero)
    assert cuda.read_device_error() == 0
    for i in range(3):
        lens = zero.clone()
        lens[i] = 1
        assert torch.equal(call(block_tables=none["block_tables"], seq_lens=lens), want)
        assert cuda.read_device_error() == 4
    assert torch.equal(call(block_tables=none["block_tables"], seq_lens=zero - 1), want)
    assert cuda.read_device_error() == 0
    # neither
    assert bool((call(**none) == 0).all()) and cuda.read_device_error() == 4
    assert bool((call(**none, seq_lens=zero, prefix_len=torch.zeros_like(p["prefix_len"])) == 0).all())
    assert cuda.read_device_error() == 0


@pytest.mark.parametrize("heads,kv_heads,dim,bs", [(8, 8, 128, 16), (32, 8, 128, 16), (8, 2, 128, 32),
                                                   (6, 2, 96, 16), (14, 2, 64, 64)])
def test_the_largest_lengths_are_cut_to_the_table(cuda, heads, kv_heads, dim, bs):
    """Lengths whose number of pages, rounded up, does not fit in 32 bits."""
    from pagedkv_fusion import ops
    p = problem(2, 100, [9, 40, 200], heads, kv_heads, dim, bs)
    p["block_tables"].clamp_(min=0)
    covered = p["block_tables"].shape[1] * bs
    decode = {k: p[k] for k in p if not k.startswith("prefix")}
    for i in range(3):
        full, huge = p["seq_lens"].clone(), p["seq_lens"].clone()
        full[i] = covered
        for n in (2 ** 31 - 1, 2 ** 31 - bs, covered + 1):
            huge[i] = n
            for call, args in ((ops.shared_prefix_attention, p), (ops.quant_paged_attention, decode)):
                want = call(**dict(args, seq_lens=full))
                assert cuda.read_device_error() == 0
                assert torch.equal(call(**dict(args, seq_lens=huge)), want), (call.__name__, i, n)
                assert cuda.read_device_error() == 4
    want = ops.shared_prefix_attention(**dict(p, prefix_len=p["prefix_len"] * 0 + len(p["prefix_table"]) * bs))
    assert torch.equal(ops.shared_prefix_attention(**dict(p, prefix_len=p["prefix_len"] * 0 + 2 ** 31 - 1)),
                       want)
    assert cuda.read_device_error() == 4
