"""Attention in 64 bits with a bound that follows from the operator's own roundings, for the
tests of weights and values far below the largest ones.

What a kernel with fp32 scores, sums and output, fp16 operands of the second product and an
fp16 result may be off, each rounding by at most half a step of its type:

* a score: D products and additions and two multiplications in fp32, each off by 2^-24 of at
  most sum|q k|/sqrt(D); a weight by that share twice (its own score's and the maximum's),
  and by 2^-22 for exp2;
* a weight (times its value's group scale, relative to the largest scale): 2^-11 of itself as a
  normal fp16 number. Below that, half of fp16's last step, 2^-25, is rounded away at most, for each of n
  positions: of weights whose largest one is held as at least 2^10, 2^-35 of it (1) times the
  value; of weights times scales, the largest of which are held as at least 2^12 and 1/2, 2^-36 of
  the largest weight times the largest value;
* values of quantized rows rounded to fp16 at half their size (v_rounded): 2^-11 of each, or
  2 * 2^-25 where fp16 has no finer step;
* the sums over n positions in fp32: 2^-24 of sum p|v| for each addition;
* the result: 2^-11 of it, or 2^-25.

Nothing in it grows with the number of positions but the fourth item and the last step's, which
stay far below the output: check() asserts that an output of zeros would fail.
"""
import math

import torch


def attend(q, k, v, seen=None, v_rounded=False):
    """q [R, D], k and v [n, D] (exact values), seen [R, n] booleans (None: all). float64 (out, bound)."""
    q, k, v = q.double(), k.double(), v.double()
    D, n = q.shape[1], k.shape[0]
    s = q @ k.T / math.sqrt(D)
    raw = q.abs() @ k.abs().T / math.sqrt(D)
    if seen is not None:
        s, raw = s.masked_fill(~seen, -math.inf), raw.masked_fill(~seen, 0)
    w = torch.exp(s - s.amax(-1, keepdim=True))
    total = w.sum(-1, keepdim=True)
    out, size = w @ v / total, w @ v.abs() / total
    e_score = 2 * (D + 4) * 2.0 ** -24 * raw.amax(-1, keepdim=True) + 2.0 ** -22
    rel = 2.0 ** -11 * (2 if v_rounded else 1) + 2.0 ** -24 * (n + 64) + e_score
    low = n * 2.0 ** -35 * v.abs().max() / total
    return out, rel * size + low + 2.0 ** -11 * out.abs() + 2.0 ** -25 + (2.0 ** -24 if v_rounded else 0.0)


def check(got, out, bound, what=""):
    assert torch.isfinite(got).all(), what
    assert (out.abs() > 4 * bound).any(-1).all(), (what, "the bound passes zeros")
    worst = float(((got.double() - out).abs() / bound).max())
    assert worst <= 1.0, (what, worst)
