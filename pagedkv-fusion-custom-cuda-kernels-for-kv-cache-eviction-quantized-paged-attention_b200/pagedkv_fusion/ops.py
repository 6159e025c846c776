"""Public operator API -- same entry points as the reference's
``pagedkv_fusion/ops.py`` (ops.py:40-141), with one execution path.

The reference dispatches to its CUDA extension when every input is a CUDA
tensor and otherwise falls back to NumPy.  Here every call runs the sm_100a
kernels of ``libpagedkv_sm100.so``:

* CUDA tensors are used in place (outputs stay on the device, work is
  enqueued on the current stream, nothing synchronizes);
* host inputs (NumPy arrays or CPU tensors) are copied to the current CUDA
  device, processed there, and the result is returned in the caller's
  container type after one device-to-host copy -- the same return types as
  the reference's fallback, without a CPU implementation behind them.

There is no CPU fallback: without the library or without a CUDA device the
call raises ``RuntimeError``.
"""

from __future__ import annotations

import math
from typing import Any

import numpy as np
import torch

try:
    from pagedkv_fusion import _C  # type: ignore[attr-defined]
    _IMPORT_ERROR: Exception | None = None
except ImportError as exc:  # pragma: no cover - exercised only without a build
    _C = None
    _IMPORT_ERROR = exc

__all__ = [
    "backend_in_use",
    "eviction_scores",
    "select_eviction_candidates",
    "eviction_scores_and_candidates",
    "EvictionPlan",
    "attention_stats",
    "quant_paged_attention",
    "DecodePlan",
    "rotary_table",
    "qk_norm_rope",
    "append_kv",
    "prefill_attention",
    "shared_prefix_attention",
    "chunk_attention",
    "accumulate_attention",
    "evict_tokens",
]


def backend_in_use() -> str:
    """'cuda' when the native library is loaded (reference ops.py:40-42)."""
    return "cuda" if _C is not None else "unavailable"


_DEVICE_OK = False


def _lib():
    global _DEVICE_OK
    if _C is None:
        raise RuntimeError(f"pagedkv_fusion native library unavailable: {_IMPORT_ERROR}")
    if not _DEVICE_OK:
        if not torch.cuda.is_available():
            raise RuntimeError("pagedkv_fusion requires a CUDA device (sm_100a); none is visible")
        _DEVICE_OK = True
    return _C


def _all_cuda(*args) -> bool:
    for a in args:
        if not (isinstance(a, torch.Tensor) and a.is_cuda):
            return False
    return True


class _Staging:
    """Moves host inputs to the current CUDA device and results back."""

    def __init__(self, *args: Any):
        self.device = next((a.device for a in args if isinstance(a, torch.Tensor) and a.is_cuda),
                           torch.device("cuda", torch.cuda.current_device()))
        self.host_kind = None
        for a in args:
            if isinstance(a, torch.Tensor) and not a.is_cuda:
                self.host_kind = self.host_kind or ("torch", a.device)
            elif not isinstance(a, torch.Tensor):
                self.host_kind = self.host_kind or ("numpy", None)

    def to_device(self, a: Any, dtype: torch.dtype | None = None) -> torch.Tensor:
        t = a if isinstance(a, torch.Tensor) else torch.from_numpy(np.ascontiguousarray(a))
        if dtype is not None and t.dtype != dtype:
            t = t.to(dtype)
        if not t.is_cuda:
            t = t.to(self.device, non_blocking=t.is_pinned())
        return t

    def back(self, t: torch.Tensor):
        if self.host_kind is None:
            return t
        # pinned destination, asynchronous copy, then wait on this stream only
        host = torch.empty(t.shape, dtype=t.dtype, pin_memory=True)
        host.copy_(t, non_blocking=True)
        torch.cuda.current_stream(t.device).synchronize()
        if self.host_kind[0] == "numpy":
            return host.numpy()
        return host


# ---------------------------------------------------------------------------
# Eviction scoring and selection
# ---------------------------------------------------------------------------

def eviction_scores(recency, frequency, attn_weights, valid_mask, w_recency: float = 0.4,
                    w_frequency: float = 0.3, w_attention: float = 0.3):
    """Fused eviction score per KV block (lower = evict first).

    Semantics of ``eviction_scores_ref`` (reference.py:38-71), bit for bit.
    """
    C = _lib()
    if _all_cuda(recency, frequency, attn_weights, valid_mask):
        return C.eviction_scores(recency, frequency, attn_weights, valid_mask, w_recency,
                                 w_frequency, w_attention)
    st = _Staging(recency, frequency, attn_weights, valid_mask)
    out = C.eviction_scores(st.to_device(recency, torch.float32),
                            st.to_device(frequency, torch.float32),
                            st.to_device(attn_weights, torch.float32),
                            st.to_device(valid_mask, torch.bool),
                            w_recency, w_frequency, w_attention)
    return st.back(out)


def select_eviction_candidates(scores, k: int):
    """Indices (int64) of the k lowest-scoring blocks, ascending by score,
    ties by lower block id (reference.py:74-81).

    Unlike the reference's GPU branch (``torch.topk``, ops.py:97-98) the tie
    order is deterministic and identical to the NumPy reference.
    """
    C = _lib()
    if _all_cuda(scores):
        return C.eviction_select(scores, int(k))
    st = _Staging(scores)
    return st.back(C.eviction_select(st.to_device(scores, torch.float32), int(k)))


def eviction_scores_and_candidates(recency, frequency, attn_weights, valid_mask, k: int,
                                   w_recency: float = 0.4, w_frequency: float = 0.3,
                                   w_attention: float = 0.3):
    """``(scores, indices)`` from one native call: the composition
    ``select_eviction_candidates(eviction_scores(...), k)``."""
    C = _lib()
    if _all_cuda(recency, frequency, attn_weights, valid_mask):
        return C.eviction_scores_select(recency, frequency, attn_weights, valid_mask, int(k),
                                        w_recency, w_frequency, w_attention)
    st = _Staging(recency, frequency, attn_weights, valid_mask)
    scores, idx = C.eviction_scores_select(st.to_device(recency, torch.float32),
                                           st.to_device(frequency, torch.float32),
                                           st.to_device(attn_weights, torch.float32),
                                           st.to_device(valid_mask, torch.bool), int(k),
                                           w_recency, w_frequency, w_attention)
    return st.back(scores), st.back(idx)


def attention_stats(k, q, sm_scale: float):
    """Per-token attention weights of a key pool for the eviction score
    (``attn_weights``): mean over KV heads of exp(s - max s) with
    s = sm_scale * q_h . K[b, t, h].  ``k`` ``[nb, bs, Hkv, 128]``, ``q``
    ``[Hkv, 128]``; returns float32 ``[nb, bs]`` in (0, 1]."""
    C = _lib()
    if _all_cuda(k, q):
        return C.attention_stats(k, q, sm_scale)
    st = _Staging(k, q)
    kd = k if isinstance(k, torch.Tensor) else torch.from_numpy(np.ascontiguousarray(k))
    return st.back(C.attention_stats(kd.to(st.device), st.to_device(q, torch.float32), sm_scale))


class EvictionPlan:
    """``eviction_scores_and_candidates`` captured once as a CUDA graph over
    fixed statistics buffers, for a serving loop that updates
    ``recency`` / ``frequency`` / ``attn_weights`` / ``valid_mask`` in place
    each step and then calls :meth:`run`.  A replay skips the per-call
    argument checks, allocations and launch of the eager call; the results
    land in the same ``scores`` / ``indices`` tensors every time.

    The buffers must be CUDA tensors that stay alive (and keep their
    storage) while the plan is used.
    """

    def __init__(self, recency, frequency, attn_weights, valid_mask, k: int,
                 w_recency: float = 0.4, w_frequency: float = 0.3, w_attention: float = 0.3):
        C = _lib()
        if not _all_cuda(recency, frequency, attn_weights, valid_mask):
            raise RuntimeError("EvictionPlan needs CUDA tensors (it binds their storage)")
        self._inputs = (recency, frequency, attn_weights, valid_mask)
        args = (recency, frequency, attn_weights, valid_mask, int(k), w_recency, w_frequency,
                w_attention)
        side = torch.cuda.Stream(device=recency.device)
        side.wait_stream(torch.cuda.current_stream(recency.device))
        with torch.cuda.stream(side):
            C.eviction_scores_select(*args)  # first call: cluster set-up, workspace sizes
        torch.cuda.current_stream(recency.device).wait_stream(side)
        self._graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self._graph):
            self.scores, self.indices = C.eviction_scores_select(*args)

    def run(self):
        """Replays the capture on the current stream; returns ``(scores, indices)``."""
        self._graph.replay()
        return self.scores, self.indices


# ---------------------------------------------------------------------------
# Quantized paged attention
# ---------------------------------------------------------------------------

def quant_paged_attention(q, k_cache_q, k_scale, v_cache_q, v_scale, block_tables, seq_lens,
                          sm_scale: float):
    """Decode-step paged attention over an INT8 paged KV cache.

    Semantics of ``paged_attention_ref`` (reference.py:140-173); fp32
    accumulation, within 1e-3 relative of the reference.
    """
    C = _lib()
    if _all_cuda(q, k_cache_q, k_scale, v_cache_q, v_scale, block_tables, seq_lens):
        return C.quant_paged_attention(q, k_cache_q, k_scale, v_cache_q, v_scale, block_tables,
                                       seq_lens, sm_scale)
    st = _Staging(q, k_cache_q, k_scale, v_cache_q, v_scale, block_tables, seq_lens)
    out = C.quant_paged_attention(st.to_device(q, torch.float32), st.to_device(k_cache_q),
                                  st.to_device(k_scale, torch.float32), st.to_device(v_cache_q),
                                  st.to_device(v_scale, torch.float32),
                                  st.to_device(block_tables, torch.int32),
                                  st.to_device(seq_lens, torch.int32), sm_scale)
    return st.back(out)


class DecodePlan:
    """``quant_paged_attention`` captured once as a CUDA graph over fixed
    buffers, for a decode loop whose batch shape stays put: each step the
    caller writes the new queries into ``q`` and the new tables / lengths
    into ``block_tables`` / ``seq_lens`` (in place), appends to the caches,
    then calls :meth:`run`.  A replay skips the argument checks, the
    workspace allocation and the host-side launch work of the eager call;
    the output lands in the same ``out`` tensor every time.

    All inputs must be contiguous CUDA tensors that keep their storage while
    the plan is used (``seq_lens`` int32).  The kernel choice is made for
    the capture's shapes; lengths up to ``block_tables``' width are
    handled by the same graph.
    """

    def __init__(self, q, k_cache_q, k_scale, v_cache_q, v_scale, block_tables, seq_lens,
                 sm_scale: float):
        C = _lib()
        bufs = (q, k_cache_q, k_scale, v_cache_q, v_scale, block_tables, seq_lens)
        if not _all_cuda(*bufs):
            raise RuntimeError("DecodePlan needs CUDA tensors (it binds their storage)")
        if not all(t.is_contiguous() for t in bufs):
            raise RuntimeError("DecodePlan needs contiguous tensors (a copy would not be rebound)")
        if q.dtype != torch.float32 or block_tables.dtype != torch.int32 or \
                seq_lens.dtype != torch.int32:
            raise RuntimeError("DecodePlan needs float32 q and int32 block_tables / seq_lens")
        self._inputs = bufs
        args = bufs + (float(sm_scale),)
        dev = q.device
        side = torch.cuda.Stream(device=dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            C.quant_paged_attention(*args)  # kernel attributes, tensor maps
        torch.cuda.current_stream(dev).wait_stream(side)
        self._graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self._graph):
            self.out = C.quant_paged_attention(*args)

    def run(self):
        """Replays the capture on the current stream; returns ``out``."""
        self._graph.replay()
        return self.out


# ---------------------------------------------------------------------------
# Rotary positions and the cache append
# ---------------------------------------------------------------------------

def rotary_table(max_positions: int, rotary_dim: int, base: float = 10000.0, scaling: str = "none",
                 factor: float = 1.0, original_positions: int = 0, beta_fast: float = 32.0,
                 beta_slow: float = 1.0, device=None) -> torch.Tensor:
    """Cosines and sines of every position, float32 ``[max_positions,
    rotary_dim]`` (``rotary_dim / 2`` cosines, then the sines), the table that
    :func:`qk_norm_rope` and :func:`append_kv` read.  Angles are taken in 64
    bits, so far positions keep their precision.

    Pair i turns by ``base ** (-2 i / rotary_dim)`` per position.  ``scaling``
    stretches a model trained on ``original_positions`` by ``factor``:

    * ``"linear"``: every frequency divided by ``factor``;
    * ``"ntk"``: ``base`` raised to ``base * factor ** (r / (r - 2))``, which
      keeps the fastest pair and divides the slowest by ``factor``;
    * ``"yarn"``: pairs that turn more than ``beta_fast`` times within
      ``original_positions`` are kept, those below ``beta_slow`` turns are
      divided by ``factor``, a linear ramp between; cosines and sines are
      multiplied by ``0.1 ln(factor) + 1``.
    """
    if max_positions < 0 or rotary_dim < 0 or rotary_dim % 2:
        raise ValueError("max_positions must be non-negative and rotary_dim even")
    if not (base > 0 and factor > 0):
        raise ValueError("base and factor must be positive")
    if device is None:
        device = torch.device("cuda", torch.cuda.current_device()) if torch.cuda.is_available() \
            else torch.device("cpu")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device)
    magnitude = 1.0
    if scaling == "ntk":
        if rotary_dim <= 2:
            raise ValueError("ntk scaling needs rotary_dim > 2")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    freq = base ** (-i / rotary_dim) if rotary_dim else i
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        if original_positions <= 0 or not beta_fast > beta_slow > 0:
            raise ValueError("yarn scaling needs original_positions > 0 and beta_fast > beta_slow")
        if factor < 1:
            raise ValueError("yarn scaling needs factor >= 1")

        def pair_of(turns):  # the (fractional) pair that turns so often in original_positions
            return rotary_dim * math.log(original_positions / (turns * 2 * math.pi)) / \
                (2 * math.log(base))

        low = max(math.floor(pair_of(beta_fast)), 0)
        high = min(math.ceil(pair_of(beta_slow)), rotary_dim - 1)
        ramp = ((i / 2 - low) / max(high - low, 1e-3)).clamp(0, 1)  # 0: kept, 1: divided
        freq = freq * (1 - ramp) + freq / factor * ramp
        magnitude = 0.1 * math.log(factor) + 1.0
    elif scaling not in ("none", "ntk"):
        raise ValueError(f"unknown scaling {scaling!r}: none, linear, ntk or yarn")
    angle = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * freq
    return (torch.cat([angle.cos(), angle.sin()], dim=1) * magnitude).float()


def qk_norm_rope(q, k, positions, rotary, q_weight=None, k_weight=None, eps: float = 1e-6,
                 interleaved: bool = False):
    """Per-head RMS norm and rotary position of queries and keys, one pass.

    ``q`` ``[T, H, D]`` and ``k`` ``[T, Hkv, D]`` (float32, float16 or
    bfloat16; ``k`` may be None) may be strided views of one projection's
    output.  With ``q_weight`` / ``k_weight`` ``[D]`` (float32 or of ``q``'s
    type) each head is divided by ``sqrt(mean(x^2) + eps)`` and multiplied by
    its weight first.  The first ``rotary.shape[1]`` channels are rotated by
    ``rotary[positions]`` (:func:`rotary_table`), as pairs ``(i, i + R/2)`` or,
    ``interleaved``, ``(2i, 2i + 1)``.  Returns new contiguous ``(q, k)``.
    The arithmetic is in 32 bits, rounded once.  A position outside the table
    gives rows of zeros and ``PKV_DEVERR_BAD_POSITION``.  No backward pass.
    """
    C = _lib()
    given = [t for t in (q, k, positions, rotary, q_weight, k_weight) if t is not None]
    if _all_cuda(*given):
        return C.qk_norm_rope(q, k, positions, rotary, q_weight, k_weight, eps, interleaved)
    st = _Staging(*given)
    q2, k2, p2, r2, qw, kw = (None if t is None else st.to_device(t)
                              for t in (q, k, positions, rotary, q_weight, k_weight))
    qo, ko = C.qk_norm_rope(q2, k2, p2, r2, qw, kw, eps, interleaved)
    return st.back(qo), None if ko is None else st.back(ko)


def append_kv(key, value, kv_cache_int8, scale_cache, slot_mapping, block_size: int,
              positions=None, rotary=None, interleaved: bool = False) -> None:
    """Appends new tokens to the paged INT8 cache in place: rotation of the
    keys (with ``positions`` and ``rotary``, as :func:`qk_norm_rope`),
    quantization and scatter in one pass on the current stream.

    ``key`` / ``value`` ``[T, Hkv, D]`` (float32, float16 or bfloat16, strided
    views allowed); ``kv_cache_int8`` ``[2, NB, bs, Hkv, D]`` and
    ``scale_cache`` ``[2, NB, Hkv]``; ``slot_mapping`` ``[T]`` with
    ``block * bs + offset``, -1 for padding.  A page whose offset 0 is written
    begins anew with the scale of its new tokens.  Otherwise the tokens below
    the lowest written offset stay: where the new tokens need a larger scale,
    their codes are moved to it, so a page filled token by token decodes as
    one filled at once, up to the rounding of each move (``write_to_cache``
    replaces the scale and leaves the codes).  Of equal slots the last token
    counts.  The caches must be CUDA tensors.  No backward pass.
    """
    _lib().append_kv(key, value, kv_cache_int8, scale_cache, slot_mapping, block_size, positions,
                     rotary, interleaved)


# ---------------------------------------------------------------------------
# Prompt attention
# ---------------------------------------------------------------------------

def prefill_attention(q, k, v, cu_seqlens, sm_scale: float, cu_seqlens_k=None,
                      causal: bool = True, return_lse: bool = False):
    """Attention over packed prompts of different lengths, grouped heads.

    ``q`` ``[total_q, H, D]``, ``k`` / ``v`` ``[total_k, Hkv, D]`` (float16 or
    bfloat16, D a multiple of 8 up to 128; strided views with contiguous
    channels are read in place); ``cu_seqlens`` int32 ``[num_seqs + 1]``, the
    sequences' first rows and the end.  ``cu_seqlens_k`` (default:
    ``cu_seqlens``) gives the keys' rows where a sequence has more keys than
    tokens, as a chunk of a longer prompt has: with ``causal``, token i of Lq
    sees keys ``j <= i + Lk - Lq``.  ``sm_scale`` > 0.

    Returns ``[total_q, H, D]`` in the inputs' type, and with ``return_lse``
    also the float32 ``[total_q, H]`` logarithms of the softmax denominators.
    Rows that see no key, and rows behind the last sequence or in front of the
    first, are zero (lse -inf).  What a row does not see does not reach it,
    whatever its value.  The probabilities are rounded to the inputs' type for
    their product with ``v``; its sums are fp32, and however long the keys a sum
    of one sign is kept to 1.1e-4.  No backward pass.
    """
    C = _lib()
    given = [t for t in (q, k, v, cu_seqlens, cu_seqlens_k) if t is not None]
    if _all_cuda(*given):
        return C.prefill_attention(q, k, v, cu_seqlens, sm_scale, cu_seqlens_k, causal, return_lse)
    st = _Staging(*given)
    got = C.prefill_attention(st.to_device(q), st.to_device(k), st.to_device(v),
                              st.to_device(cu_seqlens, torch.int32), sm_scale,
                              None if cu_seqlens_k is None else
                              st.to_device(cu_seqlens_k, torch.int32), causal, return_lse)
    return tuple(st.back(t) for t in got) if return_lse else st.back(got)


# ---------------------------------------------------------------------------
# Decode over a shared prefix
# ---------------------------------------------------------------------------

def shared_prefix_attention(q, k_cache_q, k_scale, v_cache_q, v_scale, prefix_table, prefix_len,
                            block_tables, seq_lens, sm_scale: float):
    """Decode-step attention over the INT8 paged cache for a batch whose
    sequences share a prefix (a system prompt, a document): what
    :func:`quant_paged_attention` gives for ``[prefix | own tokens]``, with
    the prefix's pages read once for the whole batch.

    ``q`` float32 ``[S, H, D]``, caches and scales as there.  ``prefix_table``
    int32 ``[P]`` and ``prefix_len`` (one integer in a tensor, read on the
    device, so a captured call follows it) give the prefix's pages;
    ``block_tables`` ``[S, M]`` and ``seq_lens`` ``[S]`` those of each
    sequence's own tokens, which start on a page of their own.  Any of the
    lengths may be 0.  D a multiple of 32 up to 128, block size up to 64.
    fp32 accuracy (root mean square of the error 1e-6 to 5e-6 of the result's).
    No backward pass.
    """
    C = _lib()
    args = (q, k_cache_q, k_scale, v_cache_q, v_scale, prefix_table, prefix_len, block_tables,
            seq_lens)
    if _all_cuda(*args):
        return C.shared_prefix_attention(*args, sm_scale)
    st = _Staging(*args)
    types = (torch.float32, None, torch.float32, None, torch.float32, torch.int32, torch.int32,
             torch.int32, torch.int32)
    return st.back(C.shared_prefix_attention(*(st.to_device(a, t) for a, t in zip(args, types)),
                                             sm_scale))


# ---------------------------------------------------------------------------
# A growing cache: new tokens' attention, their weights, eviction of tokens
# ---------------------------------------------------------------------------

def chunk_attention(q, k_cache_q, k_scale, v_cache_q, v_scale, block_tables, seq_lens, cu_seqlens,
                    sm_scale: float, return_lse: bool = False):
    """Attention of new tokens over the INT8 paged cache that holds them: one
    token of a sequence, a few drafted ones, or the next chunk of a prompt, and
    any mixture of these in one call.

    ``q`` ``[total_q, H, D]`` (float32, float16 or bfloat16; strided views with
    contiguous channels are read in place) holds the sequences' new tokens one
    behind the other, sequence s in rows ``cu_seqlens[s] .. cu_seqlens[s + 1]``
    (int32 ``[S + 1]``).  ``seq_lens`` ``[S]`` counts a sequence's tokens in the
    cache, the new ones among them (:func:`append_kv` comes first): token i of Lq
    sees the cached tokens ``j <= i + L - Lq``.  Caches, scales and tables as in
    :func:`quant_paged_attention`.  D a multiple of 32 up to 256, block size up to
    64, any group of query heads.

    Returns ``[total_q, H, D]`` in ``q``'s type, and with ``return_lse`` also the
    float32 ``[total_q, H]`` natural logarithms of the softmax denominators.  Rows
    that see no token, and rows behind the last sequence or in front of the first,
    are zero (lse -inf).  fp32 queries keep fp32 accuracy (5e-6 of the outputs' root
    mean square at any length).  With 16-bit ones the probabilities may have fp16's
    11 bits in their product with the values, which adds up to 0.8% to the error that
    rounding leaves in bf16 outputs and, for sequences of many new tokens, 43% to
    fp16's; whoever needs less passes them as fp32.  No backward pass.
    """
    C = _lib()
    args = (q, k_cache_q, k_scale, v_cache_q, v_scale, block_tables, seq_lens, cu_seqlens)
    if _all_cuda(*args):
        return C.chunk_attention(*args, sm_scale, return_lse)
    st = _Staging(*args)
    types = (None, None, torch.float32, None, torch.float32, torch.int32, torch.int32, torch.int32)
    got = C.chunk_attention(*(st.to_device(a, t) for a, t in zip(args, types)), sm_scale,
                            return_lse)
    return tuple(st.back(t) for t in got) if return_lse else st.back(got)


def accumulate_attention(weights, q, k_cache_q, k_scale, block_tables, seq_lens, cu_seqlens,
                         sm_scale: float, lse=None) -> None:
    """Adds to ``weights`` (float32 ``[NB, bs]``, one per cached token, in place)
    what the new tokens ``q`` attend to it: the sum over the tokens and the mean
    over the query heads of their softmax probabilities, so that every token
    spreads a weight of 1.

    Arguments as in :func:`chunk_attention`; ``lse`` are the log denominators that
    it returned for the same tokens, computed first where they are not given: by a
    whole pass of attention for chunks (512 tokens over 4,096: 113 us instead of 43),
    beside the weights for decode, which is faster without them (64 sequences of
    2,050 tokens: 50 us instead of 70).  At most 2^25 rows (tokens times heads).  The
    result feeds :func:`eviction_scores` as ``attn_weights`` (whole blocks) and
    :func:`evict_tokens` (single tokens); to let old weight fade, scale
    ``weights`` between calls.  A page in several tables gathers from all of them.
    The result does not depend on the order of execution.  A page that is given to
    a new sequence needs its weights zeroed.  ``weights`` must be a contiguous CUDA
    tensor, as all the others.  No backward pass.
    """
    _lib().accumulate_attention(weights, q, k_cache_q, k_scale, block_tables, seq_lens, cu_seqlens,
                                sm_scale, lse)


def evict_tokens(kv_cache_int8, scale_cache, weights, block_tables, seq_lens, keep: int,
                 sinks: int = 0, recent: int = 0):
    """Evicts single tokens from the paged INT8 cache by the weights that they
    gathered (:func:`accumulate_attention`), in place.

    A sequence of more than ``keep`` tokens keeps its first ``sinks``, its last
    ``recent`` and the heaviest of the others (of equal weights the earlier one,
    NaN heaviest), ``keep`` in all; they move, in order, to the front of its pages
    in ``kv_cache_int8`` ``[2, NB, bs, Hkv, D]``, ``scale_cache`` ``[2, NB, Hkv]``
    and ``weights`` ``[NB, bs]``.  A page takes the largest scale of the tokens it
    then holds, and codes of smaller scales are rounded to it.  Slots no longer
    used get weight 0.  Shorter sequences stay as they are.  Rotated keys keep the
    positions that they were rotated by.

    Returns ``(lens, kept)``: the new lengths, int32 ``[S]``, and the old places of
    the tokens that stayed, int32 ``[S, keep]``, ascending, then -1.  The pages
    behind the new lengths are free.  A sequence that is cut must not share pages
    with another one, nor have one twice.  CUDA tensors only.
    """
    return _lib().evict_tokens(kv_cache_int8, scale_cache, weights, block_tables, seq_lens, keep,
                               sinks, recent)
