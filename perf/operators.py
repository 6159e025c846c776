"""Cases of the prompt and shared-prefix operators: norm + rotation of queries and keys, the
append to the INT8 paged cache, attention over packed prompts, and decode over a prefix that the
whole batch shares.  ``run`` computes them in plain torch, or through ``pagedkv_fusion.ops``
where ``own`` is set."""

import glob
import math
import os
import random
import sys

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _ops():
    """The package's ``ops`` module (the package folder is not the repository's root)."""
    if "pagedkv_fusion" not in sys.modules:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, glob.glob(os.path.join(root, "pagedkv-*_b200"))[0])
    from pagedkv_fusion import ops
    return ops


def _numbers(text):
    return [int(x) for x in text.split(",")]


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------

def _text(values):
    return ",".join(str(int(v)) for v in values)


def listed():
    r = random.Random(20)
    chat = [r.randint(17, 900) for _ in range(16)]
    ragged = [r.randint(1, 256) for _ in range(64)]
    tails = [r.randint(1, 512) for _ in range(64)]
    return [
        # one short prompt at head dim 64: what counts is the latency of the call
        dict(name="prefill_short", op="prefill", q_lens="37", k_lens="37", heads=8, kv_heads=8,
             dim=64, dtype="f16", lse=False),
        # the prompts that arrived in one scheduling step, packed, GQA 32/8
        dict(name="prefill_packed", op="prefill", q_lens=_text(chat), k_lens=_text(chat), heads=32,
             kv_heads=8, dim=128, dtype="bf16", lse=False),
        # one long prompt
        dict(name="prefill_long", op="prefill", q_lens="8192", k_lens="8192", heads=32, kv_heads=8,
             dim=128, dtype="bf16", lse=False),
        # the next chunks of two long prompts: fewer queries than keys
        dict(name="prefill_chunk", op="prefill", q_lens="1000,512", k_lens="7101,4099", heads=32,
             kv_heads=8, dim=128, dtype="f16", lse=True),
        # a decode step of 64 sequences, with the norms of queries and keys
        dict(name="rope_decode", op="rope", tokens=64, heads=32, kv_heads=8, dim=128, rot=128,
             dtype="bf16", norm=True, interleaved=False, max_position=32768),
        # prompts of 16K tokens, 40/40 heads, half of each head rotated in interleaved pairs
        dict(name="rope_prompt", op="rope", tokens=16384, heads=40, kv_heads=40, dim=128, rot=64,
             dtype="f16", norm=False, interleaved=True, max_position=32768),
        # one new token for each of 64 sequences, into pages that hold earlier tokens
        dict(name="append_decode", op="append", fills=_text(1 + (i * 7) % 15 for i in range(64)),
             counts=_text([1] * 64), kv_heads=8, dim=128, bs=16, dtype="bf16", rot=128,
             interleaved=False, max_position=32768),
        # prompts of 32K tokens in all, some of which go on in a started page
        dict(name="append_prompt", op="append", fills="0,5,0,11,0,0,1,15",
             counts="8192,4001,2500,6007,333,1,3467,8268", kv_heads=8, dim=128, bs=16,
             dtype="bf16", rot=128, interleaved=False, max_position=32768),
        # eight sequences behind a short common prompt, plain heads
        dict(name="prefix_small", op="prefix", prefix=512, lens="1,2,3,5,8,13,21,32", heads=8,
             kv_heads=8, dim=128, bs=16),
        # a system prompt shared by 64 chats
        dict(name="prefix_chat", op="prefix", prefix=2040, lens=_text(ragged), heads=32,
             kv_heads=8, dim=128, bs=16),
        # a long document shared by 64 questions
        dict(name="prefix_long", op="prefix", prefix=32768, lens=_text(tails), heads=32,
             kv_heads=8, dim=128, bs=16),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _parts(rng, total, n):
    """``total`` as ``n`` positive, uneven parts."""
    cuts = sorted(rng.sample(range(1, total), n - 1)) if n > 1 else []
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


_HEADS = [(8, 8), (32, 8), (16, 2), (12, 4), (40, 40), (6, 2), (1, 1), (14, 2)]


def draw(rng):
    op = rng.choice(["prefill", "rope", "append", "prefix"])
    heads, kv = rng.choice(_HEADS)
    if op == "prefill":
        # the plain form holds heads x queries x keys scores: at most the longest prompt's
        total = _log(rng, 1, 8192)
        q_lens = _parts(rng, total, rng.randint(1, min(24, total)))
        k_lens = list(q_lens)
        if rng.random() < 0.4:
            room = 32 * 8192 * 8192 // (heads * total) - total
            k_lens = [n + rng.randint(0, max(0, min(4096, room // len(q_lens)))) for n in q_lens]
        if heads * total * sum(k_lens) > 32 * 8192 * 8192:
            heads, kv = 8, 8
        return dict(op=op, q_lens=_text(q_lens), k_lens=_text(k_lens), heads=heads, kv_heads=kv,
                    dim=rng.choice([32, 64, 80, 96, 128, 128]), dtype=rng.choice(["f16", "bf16"]),
                    lse=rng.random() < 0.3)
    if op == "rope":
        dim = rng.choice([32, 64, 80, 96, 128, 128, 256])
        return dict(op=op, tokens=_log(rng, 1, 16384 * 80 * 128 // ((heads + kv) * dim) // 4),
                    heads=heads, kv_heads=kv, dim=dim,
                    rot=rng.choice([dim, dim, dim // 2, dim // 4 // 2 * 2]),
                    dtype=rng.choice(["f32", "f16", "bf16"]), norm=rng.random() < 0.5,
                    interleaved=rng.random() < 0.5, max_position=rng.choice([4096, 32768]))
    if op == "append":
        dim, bs = rng.choice([32, 64, 96, 128, 128, 256]), rng.choice([8, 16, 16, 32, 64])
        total = _log(rng, 1, 32768 * 8 * 128 // (kv * dim) // 2)
        counts = [1] * min(total, 256) if rng.random() < 0.4 else \
            _parts(rng, total, rng.randint(1, min(24, total)))
        return dict(op=op, fills=_text(rng.choice([0, rng.randrange(bs)]) for _ in counts),
                    counts=_text(counts), kv_heads=kv, dim=dim, bs=bs,
                    dtype=rng.choice(["f32", "f16", "bf16"]), rot=rng.choice([0, dim, dim // 2]),
                    interleaved=rng.random() < 0.5, max_position=32768)
    seqs = _log(rng, 1, 96 if heads <= 16 else 48)
    top = _log(rng, 1, 512)
    return dict(op=op, prefix=_log(rng, 1, 32768 if heads <= 32 else 16384),
                lens=_text(rng.randint(0, top) for _ in range(seqs)), heads=heads, kv_heads=kv,
                dim=rng.choice([32, 64, 96, 128, 128]), bs=rng.choice([16, 16, 32]))


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _rotary(max_position, rot, dev):
    """float32 [max_position, rot]: cos | sin of the angles, taken in 64 bits."""
    freq = 10000.0 ** (-torch.arange(0, rot, 2, device=dev, dtype=torch.float64) / rot)
    angle = torch.arange(max_position, device=dev, dtype=torch.float64)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _cumulative(lens, dev):
    return torch.tensor([0] + lens, device=dev).cumsum(0).to(torch.int32)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=g, device=dev).to(dtype)

    heads, kv, dim = case.get("heads"), case["kv_heads"], case["dim"]
    s = dict(case)
    if case["op"] == "prefill":
        q_lens, k_lens = _numbers(case["q_lens"]), _numbers(case["k_lens"])
        dt = _DTYPES[case["dtype"]]
        s.update(q=normal(sum(q_lens), heads, dim, dtype=dt), k=normal(sum(k_lens), kv, dim, dtype=dt),
                 v=normal(sum(k_lens), kv, dim, dtype=dt), cu_q=_cumulative(q_lens, dev),
                 cu_k=_cumulative(k_lens, dev), same=q_lens == k_lens, scale=1.0 / math.sqrt(dim))
    elif case["op"] == "rope":
        # queries, keys and values are one projection's output: rows of (heads + 2 kv) heads
        dt, n = _DTYPES[case["dtype"]], case["tokens"]
        qkv = normal(n, heads + 2 * kv, dim, dtype=dt)
        s.update(q=qkv[:, :heads], k=qkv[:, heads:heads + kv], positions=torch.randint(
            case["max_position"], (n,), generator=g, device=dev),
            rotary=_rotary(case["max_position"], case["rot"], dev), q_weight=None, k_weight=None)
        if case["norm"]:
            s.update(q_weight=(1 + 0.1 * normal(dim)).to(dt), k_weight=(1 + 0.1 * normal(dim)).to(dt))
    elif case["op"] == "append":
        bs, dt = case["bs"], _DTYPES[case["dtype"]]
        fills, counts = _numbers(case["fills"]), _numbers(case["counts"])
        pages = [-(-(f + c) // bs) for f, c in zip(fills, counts)]
        blocks = sum(pages) + 3
        perm = torch.randperm(blocks, generator=g, device=dev)
        first = torch.tensor([0] + pages[:-1], device=dev).cumsum(0)
        count = torch.tensor(counts, device=dev)
        seq = torch.repeat_interleave(torch.arange(len(counts), device=dev), count)
        start = torch.cat([count.new_zeros(1), count.cumsum(0)[:-1]])
        at = torch.arange(sum(counts), device=dev) - start[seq] + torch.tensor(fills, device=dev)[seq]
        slots = perm[first[seq] + at // bs] * bs + at % bs
        codes = torch.randint(-127, 128, (2, blocks, bs, kv, dim), generator=g, device=dev,
                              dtype=torch.int8)
        scales = (2.0 + torch.rand((2, blocks, kv), generator=g, device=dev)) / 127
        n = sum(counts)
        s.update(key=normal(n, kv, dim, dtype=dt), value=normal(n, kv, dim, dtype=dt), cache=codes,
                 scales=scales, slots=slots, positions=None, rotary=None)
        if case["rot"]:
            s.update(positions=torch.randint(case["max_position"], (n,), generator=g, device=dev),
                     rotary=_rotary(case["max_position"], case["rot"], dev))
    else:
        bs, lens = case["bs"], _numbers(case["lens"])
        shared = -(-case["prefix"] // bs)
        pages = [-(-n // bs) for n in lens]
        blocks, width = shared + sum(pages) + 3, max(1, max(pages))
        perm = torch.randperm(blocks, generator=g, device=dev).to(torch.int32)
        tables = torch.full((len(lens), width), -1, dtype=torch.int32, device=dev)
        filled = torch.arange(width, device=dev) < torch.tensor(pages, device=dev)[:, None]
        tables[filled] = perm[shared:shared + sum(pages)]
        shape = (blocks, bs, kv, dim)
        codes = [torch.randint(-127, 128, shape, generator=g, device=dev, dtype=torch.int8)
                 for _ in range(2)]
        scales = [(2.0 + torch.rand((blocks, kv), generator=g, device=dev)) / 127 for _ in range(2)]
        s.update(q=normal(len(lens), heads, dim), k_cache=codes[0], k_scale=scales[0],
                 v_cache=codes[1], v_scale=scales[1], prefix_table=perm[:shared].clone(),
                 prefix_len=torch.tensor([case["prefix"]], dtype=torch.int32, device=dev),
                 tables=tables, seq_lens=torch.tensor(lens, dtype=torch.int32, device=dev),
                 scale=1.0 / math.sqrt(dim))
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def run(state):
    return {"prefill": _prefill, "rope": _rope, "append": _append, "prefix": _prefix}[state["op"]](state)


def _prefill(s):
    if own:
        return _ops().prefill_attention(s["q"], s["k"], s["v"], s["cu_q"], s["scale"],
                                        cu_seqlens_k=None if s["same"] else s["cu_k"],
                                        return_lse=s["lse"])
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    tq, heads, dim = q.shape
    tk, kv, _ = k.shape
    cu_q, cu_k = s["cu_q"].long(), s["cu_k"].long()
    at_q, at_k = torch.arange(tq, device=q.device), torch.arange(tk, device=q.device)
    seq_q = torch.searchsorted(cu_q[1:], at_q, right=True)
    seq_k = torch.searchsorted(cu_k[1:], at_k, right=True)
    # the last key that a query sees: its own place, counted from the sequence's end
    last = at_q - cu_q[1:][seq_q] + cu_k[1:][seq_q]
    hidden = (seq_q[:, None] != seq_k) | (at_k > last[:, None])
    rows = q.view(tq, kv, heads // kv, dim).permute(1, 2, 0, 3).reshape(kv, -1, dim)
    p = torch.bmm(rows, k.permute(1, 2, 0)).mul_(s["scale"]).view(kv, heads // kv, tq, tk)
    p.masked_fill_(hidden, -math.inf)
    m = p.amax(-1, keepdim=True)
    p.sub_(m.masked_fill(m == -math.inf, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.bmm(p.view(kv, -1, tk), v.transpose(0, 1)).view(kv, heads // kv, tq, dim)
    out = (out / total.masked_fill(total == 0, 1.0)).permute(2, 0, 1, 3).reshape(tq, heads, dim)
    out = out.to(s["q"].dtype)
    if s["lse"]:
        return out, (m + total.log()).permute(2, 0, 1, 3).reshape(tq, heads)
    return out


def _rotate(x, positions, rotary, interleaved):
    """x [T, heads, D] in 32 bits with the first rotary-width values of each head rotated."""
    rot = rotary.shape[1]
    row = rotary[positions][:, None, :]
    c, s = row[..., :rot // 2], row[..., rot // 2:]
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([y, x[..., rot:]], -1)


def _rope(s):
    if own:
        return _ops().qk_norm_rope(s["q"], s["k"], s["positions"], s["rotary"],
                                   q_weight=s["q_weight"], k_weight=s["k_weight"], eps=1e-6,
                                   interleaved=s["interleaved"])
    q, k = s["q"].float(), s["k"].float()
    if s["norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + 1e-6) * s["q_weight"].float()
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + 1e-6) * s["k_weight"].float()
    args = s["positions"], s["rotary"], s["interleaved"]
    return _rotate(q, *args).to(s["q"].dtype), _rotate(k, *args).to(s["k"].dtype)


def _values(codes, scales):
    """The cache as the values that its codes stand for, in a model's 16 bits."""
    out = torch.empty(codes.shape, dtype=torch.bfloat16, device=codes.device)
    return torch.mul(codes, scales[:, :, None, :, None], out=out)


def _append(s):
    if own:
        _ops().append_kv(s["key"], s["value"], s["cache"], s["scales"], s["slots"], s["bs"],
                         positions=s["positions"], rotary=s["rotary"],
                         interleaved=s["interleaved"])
        return _values(s["cache"], s["scales"]), s["scales"]
    key = s["key"].float()
    if s["rotary"] is not None:
        key = _rotate(key, s["positions"], s["rotary"], s["interleaved"])
    x = torch.stack([key, s["value"].float()])
    cache, scales, bs = s["cache"], s["scales"], s["bs"]
    _, blocks, _, kv, dim = cache.shape
    block, offset = s["slots"] // bs, s["slots"] % bs
    most = x.abs().amax(-1)
    index = block[None, :, None].expand_as(most)
    most = torch.zeros_like(scales).scatter_reduce(1, index, most, "amax")
    lowest = torch.full((blocks,), bs, device=x.device).scatter_reduce(0, block, offset, "amin")
    step = most / torch.full_like(most, 127.0)
    begun = (lowest == 0)[None, :, None]
    started = torch.where(step > 0, step, torch.ones_like(step))
    fresh = torch.where(begun, started, torch.maximum(scales, step))
    earlier = (torch.arange(bs, device=x.device) < lowest[:, None]) & (lowest < bs)[:, None]
    grown = (fresh > scales)[:, :, None, :, None] & earlier[None, :, :, None, None]
    moved = torch.round(cache.float() * (scales / fresh)[:, :, None, :, None])
    cache.copy_(torch.where(grown, moved, cache.float()))
    scales.copy_(fresh)
    codes = torch.round(x / fresh[:, block][..., None]).clamp(-127, 127)
    cache[:, block, offset] = codes.to(torch.int8)
    return _values(cache, scales), scales


def _prefix(s):
    if own:
        return _ops().shared_prefix_attention(s["q"], s["k_cache"], s["k_scale"], s["v_cache"],
                                              s["v_scale"], s["prefix_table"], s["prefix_len"],
                                              s["tables"], s["seq_lens"], s["scale"])
    q = s["q"]
    seqs, heads, dim = q.shape
    kv, bs, dev = s["k_cache"].shape[2], s["bs"], q.device

    def pages(cache, scale, table):  # [..., pages] -> [..., tokens, kv, dim]
        t = table.clamp(min=0).long()
        x = cache[t] * scale[t][..., None, :, None]
        return x.flatten(-4, -3)

    rows = q.view(seqs, kv, heads // kv, dim)
    shared_k = pages(s["k_cache"], s["k_scale"], s["prefix_table"])
    shared_v = pages(s["v_cache"], s["v_scale"], s["prefix_table"])
    own_k = pages(s["k_cache"], s["k_scale"], s["tables"])
    own_v = pages(s["v_cache"], s["v_scale"], s["tables"])
    by_head = rows.transpose(0, 1).reshape(kv, -1, dim)
    a = torch.bmm(by_head, shared_k.permute(1, 2, 0)).view(kv, seqs, heads // kv, -1).transpose(0, 1)
    b = torch.matmul(rows, own_k.permute(0, 2, 3, 1))
    a = a.masked_fill(torch.arange(a.shape[-1], device=dev) >= s["prefix_len"], -math.inf)
    b = b.masked_fill((torch.arange(b.shape[-1], device=dev) >=
                       s["seq_lens"][:, None])[:, None, None], -math.inf)
    p = torch.cat([a, b], -1) * s["scale"]
    p = torch.exp(p - p.amax(-1, keepdim=True))
    total = p.sum(-1, keepdim=True)
    pa, pb = p[..., :a.shape[-1]], p[..., a.shape[-1]:]
    out = torch.bmm(pa.transpose(0, 1).reshape(kv, -1, a.shape[-1]), shared_v.transpose(0, 1))
    out = out.view(kv, seqs, heads // kv, dim).transpose(0, 1)
    out = out + torch.matmul(pb, own_v.transpose(1, 2))
    return (out / total).reshape(seqs, heads, dim)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    kv, dim = case["kv_heads"], case["dim"]
    size = {"f32": 4, "f16": 2, "bf16": 2}[case.get("dtype", "f32")]
    if case["op"] == "prefill":
        q_lens, k_lens = _numbers(case["q_lens"]), _numbers(case["k_lens"])
        # query i of n sees m - n + i + 1 keys
        seen = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(q_lens, k_lens))
        rows = sum(q_lens) * case["heads"]
        return {"bytes": (2 * rows + 2 * sum(k_lens) * kv) * dim * size + 4 * rows * case["lse"],
                "flops": 4.0 * seen * case["heads"] * dim}
    if case["op"] == "rope":
        n, rows = case["tokens"], case["tokens"] * (case["heads"] + kv)
        table = min(n, case["max_position"]) * case["rot"] * 4
        return {"bytes": 2 * rows * dim * size + table + 8 * n,
                "flops": rows * (3.0 * case["rot"] + 4.0 * dim * case["norm"])}
    if case["op"] == "append":
        bs, fills, counts = case["bs"], _numbers(case["fills"]), _numbers(case["counts"])
        n, pages = sum(counts), sum(-(-(f + c) // bs) for f, c in zip(fills, counts))
        blocks = pages + 3
        values = 2 * kv * dim
        table = min(n, case["max_position"]) * case["rot"] * 4
        # keys and values in, codes out, earlier codes of started pages in and out, the scales,
        # and the whole cache as values
        return {"bytes": n * values * (size + 1) + 2 * sum(fills) * values + 16 * pages * kv +
                16 * n + table + 2 * blocks * bs * values, "flops": n * kv * (3.0 * case["rot"] + 4.0 * dim)}
    lens = _numbers(case["lens"])
    tokens = case["prefix"] + sum(lens)
    rows = case["heads"] * (case["prefix"] * len(lens) + sum(lens))
    return {"bytes": 2 * tokens * kv * dim + 8 * kv * -(-tokens // case["bs"]) +
            8 * len(lens) * case["heads"] * dim, "flops": 4.0 * rows * dim}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    def prefill(s):
        q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
        group = q.shape[1] // k.shape[1]
        out, lse = torch.zeros_like(q), q.new_full(q.shape[:2], -math.inf)
        q0 = k0 = 0
        for n, m in zip(_numbers(s["q_lens"]), _numbers(s["k_lens"])):
            seen = torch.ones(n, m, dtype=torch.bool, device=q.device).tril(m - n)
            for h in range(q.shape[1]):
                w = (q[q0:q0 + n, h] @ k[k0:k0 + m, h // group].T) * s["scale"]
                w = torch.where(seen, w, -math.inf)
                lse[q0:q0 + n, h] = torch.logsumexp(w, 1)
                out[q0:q0 + n, h] = torch.softmax(w, 1) @ v[k0:k0 + m, h // group]
            q0, k0 = q0 + n, k0 + m
        return (out, lse) if s["lse"] else out

    def turn(x, positions, rotary, interleaved):
        """Each pair as a complex number, multiplied by its unit number from the table."""
        half = rotary.shape[1] // 2
        turn = torch.complex(rotary[:, :half].double(), rotary[:, half:].double())[positions][:, None]
        x = x.clone()
        if interleaved:
            z = torch.view_as_complex(x[..., :2 * half].reshape(*x.shape[:2], half, 2)) * turn
            x[..., :2 * half] = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * turn
            x[..., :half], x[..., half:2 * half] = z.real, z.imag
        return x

    def rope(s):
        outs = []
        for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
            x = x.double()
            if w is not None:
                x = x / ((x * x).sum(-1, keepdim=True) / x.shape[-1] + 1e-6).sqrt() * w.double()
            outs.append(turn(x, s["positions"], s["rotary"], s["interleaved"]))
        return tuple(outs)

    def append(s):
        key = s["key"].double()
        if s["rotary"] is not None:
            key = turn(key, s["positions"], s["rotary"], s["interleaved"])
        x = torch.stack([key, s["value"].double()])
        bs = s["bs"]
        _, blocks, _, kv, dim = s["cache"].shape
        # the call's tokens laid out as pages, with what was in them
        block, offset = s["slots"] // bs, s["slots"] % bs
        new = x.new_zeros(2, blocks, bs, kv, dim)
        new[:, block, offset] = x
        written = torch.zeros(blocks, bs, dtype=torch.bool, device=x.device)
        written[block, offset] = True
        touched = written.any(1)
        lowest = written.int().argmax(1)
        old = s["scales"].double()
        step = new.abs().amax((2, 4)) / 127
        fresh = torch.where(lowest[:, None] == 0, torch.where(step > 0, step, 1.0), torch.maximum(old, step))
        scale = torch.where(touched[:, None], fresh, old)
        codes = s["cache"].double()
        before = (torch.arange(bs, device=x.device) < lowest[:, None]) & touched[:, None]
        again = torch.round(codes * (old / scale)[:, :, None, :, None])
        codes = torch.where(before[None, :, :, None, None], again, codes)
        fit = torch.round(new / scale[:, :, None, :, None]).clamp(-127, 127)
        codes = torch.where(written[None, :, :, None, None], fit, codes)
        return codes * scale[:, :, None, :, None], scale

    def prefix(s):
        q = s["q"].double()
        group, bs = q.shape[1] // s["k_cache"].shape[2], s["bs"]
        out = torch.zeros_like(q)
        lens = _numbers(s["lens"])

        def tokens(cache, scale, pages, n, h):
            pages = pages.long()
            return (cache[pages, :, h].double() * scale[pages, h].double()[:, None, None]).flatten(0, 1)[:n]

        for h in range(s["k_cache"].shape[2]):
            heads = slice(h * group, (h + 1) * group)
            front = [tokens(c, f, s["prefix_table"], s["prefix"], h) for c, f in
                     ((s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"]))]
            for i, n in enumerate(lens):
                mine = s["tables"][i, :-(-n // bs)]
                k = torch.cat([front[0], tokens(s["k_cache"], s["k_scale"], mine, n, h)])
                v = torch.cat([front[1], tokens(s["v_cache"], s["v_scale"], mine, n, h)])
                out[i, heads] = torch.softmax(q[i, heads] @ k.T * s["scale"], -1) @ v
        return out

    return {"prefill": prefill, "rope": rope, "append": append, "prefix": prefix}[case["op"]](
        prepare(case, seed))
