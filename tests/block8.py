"""A cache in e4m3 codes with a scale for each block of positions and head, and the position
rotation, in 64 bits on any device: what the tests of va_attend_paged and va_append_rope
compare with."""
import math

import torch

E4M3 = torch.float8_e4m3fn


def need(top):
    """The smallest power of two in [2^-24, 2^15] whose 448-fold is not below top (float64)."""
    top = top.double()
    e = torch.ceil(torch.log2(top.clamp(min=2.0 ** -40) / 448))
    e = torch.where(448 * torch.exp2(e - 1) >= top, e - 1, e)
    e = torch.where(448 * torch.exp2(e) < top, e + 1, e)
    return torch.exp2(e.clamp(-24, 15))


def codes(x, s):
    """e4m3 codes (uint8) of x / s, float64, nearest even, at most 448, NaN for what is not finite."""
    q = torch.where(x.isfinite(), (x / s).clamp(-448, 448), torch.full_like(x, math.nan))
    return q.float().to(E4M3).view(torch.uint8)          # float() moves no value over a border of 4 bits unless it is within 2^-25 of it


def pack(x, G):
    """rows [.., n, D] (n a multiple of G) -> codes (float8) and fp16 scales [.., n / G]."""
    y = x.double().unflatten(-2, (-1, G))
    s = need(y.abs().amax((-1, -2)))
    return codes(y, s[..., None, None]).flatten(-3, -2).view(E4M3), s.half()


def values(pool, scales):
    """float64 rows [num_pages, Hkv, page_rows, D] of a pool."""
    G = pool.shape[2] // scales.shape[2]
    return pool.view(torch.uint8).view(E4M3).double() * scales.double().abs().repeat_interleave(G, 2)[..., None]


def rows(vals, table, n, h):
    """Positions 0 .. n - 1 of a sequence's head: vals as values() gives them, table its pages."""
    page_rows = vals.shape[2]
    p = torch.arange(n, device=vals.device)
    return vals[torch.as_tensor(table, device=vals.device).long()[p // page_rows], h, p % page_rows]


def rotate(x, places, freq, interleaved, scaling=1.0):
    """x [T, H, D], places [T], freq [R / 2] (float32): float64 rotated rows, and a bound of what a
    kernel may be off before it rounds its result: cos and sin of an angle in turns as fp32 (off by half
    of 2^-25, 2 pi times that as an angle), each off by 2^-22.9 by the instruction, their product with the
    scaling, and two products and an addition in fp32: together below 2^-21 of |x| + |y|, scaled."""
    x, R = x.double().clone(), 2 * freq.numel()
    t = places.double()[:, None, None] * freq.double()
    c, s = t.cos() * scaling, t.sin() * scaling
    a, b = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    p, q = x[..., a].clone(), x[..., b].clone()
    x[..., a], x[..., b] = p * c - q * s, p * s + q * c
    off = torch.zeros_like(x)
    off[..., a] = off[..., b] = (p.abs() + q.abs()) * abs(scaling) * 2.0 ** -21
    return x, off
