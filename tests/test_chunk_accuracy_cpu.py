"""The accuracy that chunk_attention and accumulate_attention are built for with float32 queries, as
limits that a loss of precision does not pass, and models of the kernels' arithmetic that show so:
whole, they are within the limits; with one of their parts left out, they are not.

The errors are root mean squares over those of what is wanted, for V codes of one sign, so that an
error that always has one sign shows too.  Scores have a standard deviation of SPREAD.

* Outputs: what the tensor cores cut of O between two flushes of it (test_prefix_accuracy_cpu.py: 16
  keys lose 1.2 / 2 * 0.7 * 2^-23 of a sum that grows evenly), 4.0e-6 for 5 tiles of 128 keys
  (sequences of many rows), 3.2e-6 for 512 keys (of few rows), and 1e-6 of either sign: 5e-6.
* Log denominators and gathered weights: a score is a sum of D / 16 steps for each half of the query,
  which is cut by up to a last place, 2^-23, of the largest sum on the way.  Where codes come 128 too
  large that is 256 sum(q), 3.5 times a score's deviation: in the mean of a step half of
  2^-23 * 3.5 * 2.5 nats, 5.2e-7, over D / 8 steps 8.3e-6 (D = 128), 1.7e-5 (D = 256).  It
  has one sign for a row's keys, so it shows in the denominator and, where that was summed in another
  order, in the weights.  Denominators add half a step of their own, 2^-21 at 16 to 32: 1e-5 and 2e-5.
  A query without its lower half is off by 2^-12.2 of a score's deviation, 5e-4 nats, each key on its
  own, which the sum over a weight's rows that count, or a denominator's keys, shrinks by their root:
  more than 4e-5 where these are up to 100.
"""

from __future__ import annotations

import numpy as np
import pytest

from test_prefix_accuracy_cpu import SPREAD, cut, error, exact, halves, inputs, model, step

TILES = 5                      # of 128 keys between two flushes, many rows
KEYS = 512                     # keys between two flushes, few rows
LIMIT = 5e-6                   # outputs
SCORE_LIMIT = {128: 1e-5, 256: 2e-5}  # weights and log denominators, by head_dim

LOG2E = 1.4426950408889634


def row_powers(q):
    return (2.0 ** (10 - np.floor(np.log2(np.abs(q).max(1, keepdims=True))))).astype(np.float32)


def scores_of_rows(x, q_low=True):
    """Scores in powers of two as the kernel of few rows takes them: codes 128 too large."""
    q, dim, up = x["q"], x["q"].shape[1], row_powers(x["q"])
    hi, lo = halves((q * up).astype(np.float32), q_low)
    k = x["k"] + 128.0
    sums = []
    for part, start in ((hi, -128.0 * (hi.sum(1) + lo.sum(1))), (lo, np.zeros(len(q)))):
        s = np.repeat(start.astype(np.float32).astype(np.float64)[:, None], len(k), 1)
        for c in range(0, dim, 16):
            s = cut(s + part[:, c:c + 16] @ k[:, c:c + 16].T)
        sums.append(s.astype(np.float32))
    f = ((1 / up) * np.float32(x["scale"] * LOG2E)).astype(np.float32)
    return ((sums[0] + sums[1]).astype(np.float32) * (x["k_scale"] * f).astype(np.float32)).astype(np.float32)


def rows_model(x, keys, q_low=True, p_low=True):
    """Few rows, one warp over all keys: steps of 16, the lower halves first."""
    f32 = np.float32
    y, v = scores_of_rows(x, q_low), x["v"]
    unit = f32(2.0 ** np.ceil(np.log2(x["v_scale"].max())))
    vr = x["v_scale"] / unit
    n = len(y)
    base, most = np.zeros((n, 1), f32), np.full((n, 1), -np.inf, f32)
    l, total_l = np.zeros((n, 1), f32), np.zeros((n, 1), f32)
    O, total = np.zeros((n, v.shape[1])), np.zeros((n, v.shape[1]), f32)
    for j in range(0, len(v), 16):
        at = slice(j, j + 16)
        if keys and j and j % keys == 0:
            total, total_l = (total + O).astype(f32), total_l + l
            O, l = np.zeros_like(O), np.zeros_like(l)
        top = y[:, at].max(1, keepdims=True)
        move = top > most
        to = (top - f32(13)).astype(f32)
        a = np.where(move, np.where(np.isinf(most), 0, np.exp2(np.minimum(base - to, 0))), 1).astype(f32)
        base, most = np.where(move, to, base), np.where(move, top + f32(2), most)
        O, l = (O * a).astype(f32).astype(np.float64), l * a
        total, total_l = total * a, total_l * a  # (the kernel does that when it adds them)
        p = np.exp2((y[:, at] - base).astype(f32).astype(np.float64)).astype(f32)
        l = l + p.sum(1, keepdims=True, dtype=f32)
        hi, lo = halves((p * vr[at]).astype(f32), p_low)
        for part in (lo, hi):
            O = step(O, part, v[at])
    return (total + O) * unit / (total_l + l)


@pytest.mark.parametrize("tokens", [2432, 4736])
def test_the_limit_of_outputs_holds_and_tells_a_loss(tokens):
    x = inputs(tokens, tokens)
    want = exact(x)
    for kernel, often in ((model, TILES), (rows_model, KEYS)):
        assert error(kernel(x, often), want) <= LIMIT
        assert error(kernel(x, often, q_low=False), want) > LIMIT
        assert error(kernel(x, often, p_low=False), want) > LIMIT
        assert error(kernel(x, None), want) > LIMIT


@pytest.mark.parametrize("dim", [128, 256])
def test_the_limit_of_scores_holds_and_tells_a_loss(dim):
    x = inputs(dim, 3000, rows=96, dim=dim)
    s = x["q"].astype(np.float64) @ (x["k"] * x["k_scale"][:, None]).T * x["scale"]
    assert 0.7 * SPREAD < s.std() < 1.4 * SPREAD
    lse = np.log(np.exp(s).sum(1))
    want = np.exp(s - lse[:, None]).sum(0)
    for q_low in (True, False):
        y = scores_of_rows(x, q_low).astype(np.float64)
        got_lse = np.log(np.exp2(y).sum(1))
        got = np.exp2(y - (lse.astype(np.float32) * np.float32(LOG2E))[:, None]).astype(np.float32).sum(0)
        within = (error(got, want) <= SCORE_LIMIT[dim],
                  float(np.sqrt(np.mean((got_lse - lse) ** 2))) <= SCORE_LIMIT[dim])
        assert within == (q_low, q_low)
