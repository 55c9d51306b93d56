"""Attention in 64 bits with a derived error bound, for the prompt and tree kernels' tests.

The bound counts what a kernel with fp32 scores, sums and output, fp16 weights and an fp16
result may be off, each rounding by at most half a step of its type:

* a score is a sum of D exact products in fp32: each of its additions and the multiplications
  by a group's scale and by log2(e)/sqrt(D) is off by 2^-24 of at most sum|q k|/sqrt(D), so a
  weight is off by that share twice (its own score's and the maximum's), and by 2^-22 for exp2;
* a weight (times V's group scale) is rounded to fp16: 2^-11 of it, or 2^-25 absolutely where
  fp16 has no finer step, in units of the largest weight, which is at least 1;
* where a kernel rounds V's values to fp16 (v_rounded: code times scale, a product of 8 and 11 bits,
  in 11), each is off by 2^-11 of itself, the sum of weights times values by 2^-11 of sum p|v| more;
* the sums over n positions are off by 2^-24 of sum p|v| for each addition;
* the result is rounded to fp16: 2^-11 of it, or 2^-25.
"""
import math

import torch


def attend(q, k, v, seen, scale_v=None, v_rounded=False):
    """q [R, D], k and v [n, D] (exact values), seen [R, n] booleans; scale_v [n, D]: the group scale
    under each value of v (1 where there are none). float64 (out, bound), zeros where nothing is seen."""
    q, k, v = q.double(), k.double(), v.double()
    D, n = q.shape[1], k.shape[0]
    if n == 0:
        return torch.zeros_like(q), torch.zeros_like(q)
    s = (q @ k.T / math.sqrt(D)).masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    w = torch.exp(s - top.masked_fill(top == -math.inf, 0))
    total = w.sum(-1, keepdim=True)
    total = total.masked_fill(total == 0, 1)
    out, size = w @ v / total, w @ v.abs() / total
    raw = (q.abs() @ k.abs().T / math.sqrt(D)).masked_fill(~seen, 0).amax(-1, keepdim=True)
    e_score = 2 * (D + 4) * 2.0 ** -24 * raw + 2.0 ** -22
    sv = torch.ones_like(v) if scale_v is None else scale_v.double()
    code = torch.where(sv == 0, torch.zeros_like(v), v / sv).abs()
    fine = seen.double() @ code * 2.0 ** -25 / total                 # weights below fp16's smallest normal one
    bound = (2.0 ** -11 * (2 if v_rounded else 1) + 2.0 ** -24 * (n + 64) + e_score) * size + fine + 2.0 ** -11 * out.abs() + 2.0 ** -25
    return out, bound


def check(got, out, bound, what=""):
    off = (got.double() - out).abs()
    assert torch.isfinite(got).all(), what
    worst = float((off / bound).max()) if out.numel() else 0.0
    assert worst <= 1.0, (what, worst)
    return worst
