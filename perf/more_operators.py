"""Cases of the operators on a growing INT8 cache: attention of new tokens (one, a few, or a
prompt's next chunk) over the paged cache, the accumulation of their attention weights per cached
token, and the eviction of the tokens that gathered least.  ``run`` computes them in plain torch,
or through ``pagedkv_fusion.ops`` where ``own`` is set."""

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
    r = random.Random(5)
    ragged = [r.randint(1200, 2900) for _ in range(64)]
    drafts = [r.randint(1, 8) for _ in range(24)]
    behind = [n + r.randint(100, 4000) for n in drafts]
    grown = [r.randint(1500, 2600) for _ in range(64)]
    return [
        # one short prompt of float32 heads, all of it new: what counts is the latency of the call
        dict(name="chunk_small", op="chunk", q_lens="37", lens="37", heads=8, kv_heads=8, dim=64,
             bs=16, dtype="f32", lse=False),
        # a decode step of 64 sequences with 16-bit queries
        dict(name="chunk_decode", op="chunk", q_lens=_text([1] * 64), lens=_text(ragged), heads=32,
             kv_heads=8, dim=128, bs=16, dtype="bf16", lse=True),
        # drafted tokens of 24 sequences, verified together
        dict(name="chunk_verify", op="chunk", q_lens=_text(drafts), lens=_text(behind), heads=32,
             kv_heads=8, dim=128, bs=16, dtype="f16", lse=False),
        # a scheduling step: the next chunk of one prompt beside seven decoding sequences
        dict(name="chunk_mixed", op="chunk", q_lens="1,1,512,1,1,1,1,1",
             lens="801,1502,3333,40,2777,1200,4000,599", heads=32, kv_heads=8, dim=128, bs=32,
             dtype="bf16", lse=False),
        # the last chunk of a long prompt
        dict(name="chunk_prompt", op="chunk", q_lens="2048", lens="16384", heads=32, kv_heads=8,
             dim=128, bs=16, dtype="bf16", lse=True),
        # statistics of eight short sequences of a float32 model
        dict(name="weights_small", op="weights", q_lens=_text([1] * 8), lens="9,200,33,64,1,128,77,150",
             heads=8, kv_heads=8, dim=64, bs=16, dtype="f32", lse=False),
        # the statistics of a decode step of 64 sequences, the log denominators not at hand
        dict(name="weights_decode", op="weights", q_lens=_text([1] * 64), lens=_text(ragged),
             heads=32, kv_heads=8, dim=128, bs=16, dtype="bf16", lse=False),
        # a prompt's last 64 tokens look back over all of it, after their attention
        dict(name="weights_window", op="weights", q_lens="64", lens="32768", heads=32, kv_heads=8,
             dim=128, bs=16, dtype="bf16", lse=True),
        # three sequences, one of them short enough to stay
        dict(name="evict_small", op="evict", lens="300,100,251", keep=128, sinks=4, recent=32,
             kv_heads=8, dim=64, bs=16),
        # 64 sequences that have grown to twice their share are cut back
        dict(name="evict_batch", op="evict", lens=_text(grown), keep=1024, sinks=4, recent=256,
             kv_heads=8, dim=128, bs=16),
        # a long prompt is cut to its heaviest tokens before decoding
        dict(name="evict_long", op="evict", lens="32768", keep=4096, sinks=16, recent=64,
             kv_heads=8, dim=128, bs=32),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


_HEADS = [(8, 8), (32, 8), (16, 2), (12, 4), (40, 40), (6, 2), (1, 1), (14, 2)]


def draw(rng):
    op = rng.choice(["chunk", "weights", "evict"])
    heads, kv = rng.choice(_HEADS)
    dim, bs = rng.choice([32, 64, 96, 128, 128]), rng.choice([8, 16, 16, 32, 64])
    if op == "evict":
        seqs = _log(rng, 1, 64)
        top = _log(rng, 16, max(16, min(32768, 64 * 2048 * 1024 // (seqs * max(kv * dim, 512)))))
        keep = rng.randint(1, top)
        sinks = rng.randint(0, min(16, keep))
        return dict(op=op, lens=_text(rng.randint(max(1, top // 2), top) for _ in range(seqs)),
                    keep=keep, sinks=sinks, recent=rng.randint(0, keep - sinks), kv_heads=kv,
                    dim=dim, bs=bs)
    seqs, most = {"decode": (_log(rng, 1, 64), 1), "verify": (_log(rng, 1, 32), 8),
                  "prompt": (rng.randint(1, 4), _log(rng, 9, 2048))}[
        rng.choice(["decode", "verify", "prompt"])]
    q_lens = [rng.randint(1, most) for _ in range(seqs)]
    # the plain form holds the scores of the longest chunk and sequence for all of them, and the
    # cache as values
    room = min(2048 * 16384 * 32 // (seqs * heads * most), 64 * 2900 * 8 * 128 // (seqs * kv * dim),
               16384)
    top = _log(rng, 1, max(1, room))
    return dict(op=op, q_lens=_text(q_lens), lens=_text(n + rng.randint(top // 2, top) for n in q_lens),
                heads=heads, kv_heads=kv, dim=dim, bs=bs, dtype=rng.choice(["f32", "f16", "bf16"]),
                lse=rng.random() < 0.5)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    kv, dim, bs, lens = case["kv_heads"], case["dim"], case["bs"], _numbers(case["lens"])
    pages = [-(-n // bs) for n in lens]
    blocks, width = sum(pages) + 3, max(pages)
    perm = torch.randperm(blocks, generator=g, device=dev).to(torch.int32)
    tables = torch.full((len(lens), width), -1, dtype=torch.int32, device=dev)
    filled = torch.arange(width, device=dev) < torch.tensor(pages, device=dev)[:, None]
    tables[filled] = perm[:sum(pages)]
    codes = torch.randint(-127, 128, (2, blocks, bs, kv, dim), generator=g, device=dev,
                          dtype=torch.int8)
    scales = (2.0 + torch.rand((2, blocks, kv), generator=g, device=dev)) / 127
    s = dict(case, cache=codes, scales=scales, tables=tables,
             seq_lens=torch.tensor(lens, dtype=torch.int32, device=dev))
    if case["op"] == "evict":
        # a few tokens gather most of the weight
        s.update(stats=torch.rand((blocks, bs), generator=g, device=dev).pow(8),
                 weights=torch.empty(blocks, bs, device=dev))
        return s
    q_lens = _numbers(case["q_lens"])
    q = torch.randn((sum(q_lens), case["heads"], dim), generator=g, device=dev)
    s.update(q=q.to(_DTYPES[case["dtype"]]), scale=1.0 / math.sqrt(dim), most=max(q_lens),
             cu=torch.tensor([0] + q_lens, device=dev).cumsum(0).to(torch.int32))
    if case["op"] == "weights":
        s.update(weights=torch.rand((blocks, bs), generator=g, device=dev), given=None)
        if case["lse"]:  # what the attention of the same tokens gave
            p, total, m, there, _ = _scores(s)
            s["given"] = _rows(m + total.log(), there)[..., 0].contiguous()
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def run(state):
    return {"chunk": _chunk, "weights": _weights, "evict": _evict}[state["op"]](state)


def _tokens(codes, scales, tables):
    """The sequences' tokens as values in 32 bits, [sequence, head, token, channel]."""
    t = tables.clamp(min=0).long()
    x = codes[t] * scales[t][..., None, :, None]
    return x.flatten(1, 2).transpose(1, 2)


def _scores(s):
    """exp(score - max) of every sequence's new tokens over its cached ones, padded to the longest:
    [sequence, kv head, head of the group, token, key]; the sums and maxima over the keys; which
    tokens there are, and their rows."""
    q, cu, length = s["q"].float(), s["cu"].long(), s["seq_lens"].long()
    seqs, kv, dev = len(length), s["kv_heads"], q.device
    count, at = cu[1:] - cu[:-1], torch.arange(s["most"], device=dev)
    there = at < count[:, None]
    row = torch.where(there, cu[:-1, None] + at, 0)
    x = q[row].view(seqs, s["most"], kv, -1, s["dim"]).permute(0, 2, 3, 1, 4)
    k = _tokens(s["cache"][0], s["scales"][0], s["tables"])
    p = torch.matmul(x.flatten(2, 3), k.transpose(-1, -2)).mul_(s["scale"])
    p = p.view(seqs, kv, -1, s["most"], k.shape[2])
    # a token sees the keys up to its own place, counted from the sequence's end
    last = torch.minimum(at + (length - count)[:, None], length[:, None] - 1)
    hidden = torch.arange(k.shape[2], device=dev) > last[..., None]
    p.masked_fill_(hidden[:, None, None], -math.inf)
    m = p.amax(-1, keepdim=True)
    p.sub_(m.masked_fill(m == -math.inf, 0.0)).exp_()
    return p, p.sum(-1, keepdim=True), m, there, row


def _rows(x, there):
    """[sequence, kv head, head of the group, token, n] to [token of the batch, head, n]."""
    return x.permute(0, 3, 1, 2, 4).flatten(2, 3)[there]


def _chunk(s):
    if own:
        return _ops().chunk_attention(s["q"], s["cache"][0], s["scales"][0], s["cache"][1],
                                      s["scales"][1], s["tables"], s["seq_lens"], s["cu"],
                                      s["scale"], return_lse=s["lse"])
    p, total, m, there, _ = _scores(s)
    v = _tokens(s["cache"][1], s["scales"][1], s["tables"])
    x = torch.matmul(p.flatten(2, 3), v).view(*p.shape[:4], -1)
    out = _rows(x / total.masked_fill(total == 0, 1.0), there).to(s["q"].dtype)
    return (out, _rows(m + total.log(), there)[..., 0]) if s["lse"] else out


def _weights(s):
    if own:
        _ops().accumulate_attention(s["weights"], s["q"], s["cache"][0], s["scales"][0],
                                    s["tables"], s["seq_lens"], s["cu"], s["scale"], lse=s["given"])
        return s["weights"]
    p, total, m, there, row = _scores(s)
    if s["given"] is not None:
        total = s["given"][row].view(*row.shape, s["kv_heads"], -1).permute(0, 2, 3, 1)[..., None]
        total = torch.exp(total - m)
    p = (p / total.masked_fill(total == 0, 1.0)).mul_(there[:, None, None, :, None])
    most = p.sum((1, 2, 3)) / s["heads"]
    bs, at = s["bs"], torch.arange(most.shape[1], device=most.device)
    seen = at < s["seq_lens"][:, None]
    slots = (s["tables"].long() * bs).repeat_interleave(bs, 1) + at % bs
    s["weights"].view(-1).index_add_(0, slots[seen], most[seen])
    return s["weights"]


def _values(codes, scales):
    """The cache as the values that its codes stand for, in a model's 16 bits."""
    out = torch.empty(codes.shape, dtype=torch.bfloat16, device=codes.device)
    return torch.mul(codes, scales[:, :, None, :, None], out=out)


def _evict(s):
    s["weights"].copy_(s["stats"])  # what the steps since the last eviction have gathered
    cache, scales, weights, keep, bs = s["cache"], s["scales"], s["weights"], s["keep"], s["bs"]
    if own:
        lens, kept = _ops().evict_tokens(cache, scales, weights, s["tables"], s["seq_lens"], keep,
                                         sinks=s["sinks"], recent=s["recent"])
        return _values(cache, scales), scales, weights, lens, kept
    length = s["seq_lens"].long()[:, None]
    at = torch.arange(s["tables"].shape[1] * bs, device=cache.device).expand(len(length), -1)
    there = at < length
    slots = (s["tables"].long() * bs).repeat_interleave(bs, 1) + at % bs
    rank = torch.where(there, weights.view(-1)[slots.clamp(min=0)], -math.inf)
    rank = rank.masked_fill(there & ((at < s["sinks"]) | (at >= length - s["recent"])), math.inf)
    order = rank.sort(dim=1, descending=True, stable=True).indices[:, :keep]
    stays = torch.zeros_like(there).scatter(1, order, True) & there
    lens = stays.sum(1)
    to = stays.cumsum(1) - 1
    kept = torch.full((len(length), keep), -1, dtype=torch.int32, device=cache.device)
    seq = torch.arange(len(length), device=cache.device)[:, None].expand_as(at)[stays]
    kept[seq, to[stays]] = at[stays].int()
    source, target = slots[stays], slots[seq, to[stays]]
    old = scales[:, source // bs]
    fresh = torch.full_like(scales, -math.inf).index_reduce_(1, target // bs, old, "amax")
    new = fresh[:, target // bs]
    codes = cache.flatten(1, 2)[:, source].float()
    moved = torch.round(codes * (old / new)[..., None]).clamp(-127, 127)
    codes = torch.where((old < new)[..., None], moved, codes)
    cache.flatten(1, 2)[:, target] = codes.to(torch.int8)
    scales.copy_(torch.where(fresh > -math.inf, fresh, scales))
    gathered = weights.view(-1)[source]
    weights.view(-1)[slots[there]] = 0.0
    weights.view(-1)[target] = gathered
    return _values(cache, scales), scales, weights, lens.int(), kept


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    kv, dim, bs, lens = case["kv_heads"], case["dim"], case["bs"], _numbers(case["lens"])
    pages = sum(-(-n // bs) for n in lens)
    if case["op"] == "evict":
        cut = [n for n in lens if n > case["keep"]]
        moved = len(cut) * case["keep"]
        blocks = pages + 3
        # kept codes in and out with their pages' scales, the statistics in and out, what was
        # kept, and the whole cache as values
        return {"bytes": 4 * moved * kv * dim + 32 * kv * moved // bs + 8 * sum(cut) +
                4 * len(lens) * (2 + case["keep"]) + 4 * blocks * bs * kv * dim,
                "flops": 2.0 * moved * kv * dim}
    q_lens, heads = _numbers(case["q_lens"]), case["heads"]
    size = {"f32": 4, "f16": 2, "bf16": 2}[case["dtype"]]
    # new token i of n sees m - n + i + 1 cached ones
    seen = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(q_lens, lens))
    rows, tokens = sum(q_lens) * heads, sum(lens)
    if case["op"] == "weights":
        return {"bytes": rows * dim * size + tokens * kv * dim + 4 * pages * (kv + 1) + 8 * tokens +
                4 * rows * case["lse"], "flops": 2.0 * seen * heads * dim}
    return {"bytes": 2 * rows * dim * size + 2 * tokens * kv * dim + 4 * pages * (2 * kv + 1) +
            4 * rows * case["lse"], "flops": 4.0 * seen * heads * dim}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    bs, lens = s["bs"], _numbers(s["lens"])

    def head(kind, pages, n, h):
        """The values of a sequence's tokens, one head."""
        pages = pages.long()
        x = s["cache"][kind, pages, :, h].double() * s["scales"][kind, pages, h].double()[:, None, None]
        return x.flatten(0, 1)[:n]

    if case["op"] == "evict":
        keep, sinks, recent = s["keep"], s["sinks"], s["recent"]
        codes, scales, weights = s["cache"].double(), s["scales"].double(), s["stats"].double()
        out_lens, out_kept = [], torch.full((len(lens), keep), -1, dtype=torch.int32)
        for i, n in enumerate(lens):
            pages = s["tables"][i, :-(-n // bs)].long()
            if n <= keep:
                out_lens.append(n)
                out_kept[i, :n] = torch.arange(n)
                continue
            w = weights[pages].flatten()[:n]
            middle = w[sinks:n - recent]
            # ties go to the lower index: a stable sort of the negated weights
            best = torch.sort(-middle, stable=True).indices[:keep - sinks - recent].sort().values
            kept = torch.cat([torch.arange(sinks, device=w.device), best + sinks,
                              torch.arange(n - recent, n, device=w.device)])
            out_lens.append(keep)
            out_kept[i] = kept.cpu().int()
            old_codes = codes[:, pages].flatten(1, 2)[:, kept]
            old_scale = scales[:, pages[kept // bs]]
            for j in range(-(-keep // bs)):  # page by page
                part = slice(j * bs, min((j + 1) * bs, keep))
                size = part.stop - part.start
                new = old_scale[:, part].amax(1)
                ratio = old_scale[:, part] / new[:, None]
                codes[:, pages[j], :size] = torch.where(
                    ratio[..., None] < 1, torch.round(old_codes[:, part] * ratio[..., None]),
                    old_codes[:, part])
                scales[:, pages[j]] = new
            flat = torch.cat([w[kept], w.new_zeros(n - keep)])
            full = weights[pages].flatten()
            full[:n] = flat
            weights[pages] = full.view(-1, bs)
        return (codes * scales[:, :, None, :, None], scales, weights,
                torch.tensor(out_lens, dtype=torch.int32), out_kept)

    q, q_lens = s["q"].double(), _numbers(s["q_lens"])
    group = s["heads"] // s["kv_heads"]
    out, lse = torch.zeros_like(q), q.new_full(q.shape[:2], -math.inf)
    total = s["weights"].double() if case["op"] == "weights" else None
    at = 0
    for i, (n, m) in enumerate(zip(q_lens, lens)):
        pages = s["tables"][i, :-(-m // bs)]
        seen = torch.ones(n, m, dtype=torch.bool, device=q.device).tril(m - n)
        gathered = q.new_zeros(pages.numel() * bs)
        for h in range(s["kv_heads"]):
            k = head(0, pages, m, h)
            v = head(1, pages, m, h) if total is None else None
            for a in range(h * group, (h + 1) * group):
                w = torch.where(seen, q[at:at + n, a] @ k.T * s["scale"], -math.inf)
                lse[at:at + n, a] = torch.logsumexp(w, 1)
                if total is None:
                    out[at:at + n, a] = torch.softmax(w, 1) @ v
                else:
                    gathered[:m] += torch.softmax(w, 1).sum(0) / s["heads"]
        if total is not None:
            total[pages.long()] += gathered.view(-1, bs)
        at += n
    if total is not None:
        return total
    return (out, lse) if s["lse"] else out
