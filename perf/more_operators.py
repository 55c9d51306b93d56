"""The block-scaled 8-bit cache as measurable cases: what writes it and what reads it.

* ``append``: the rows of a projection (q, k and v as slices of it) rotated by their
  positions, k and v written into the paged cache, in 8 bits with a scale for each block of
  positions and head or as fp16, q (and k) returned (``append_rope``);
* ``attend``: attention of each sequence's newest tokens, one or many, over its cache in 8
  bits, causal among themselves (``attend_paged``).

The plain forms are elementary torch operations in fp32, angles in fp64. Activations are
N(0, 1) draws; caches hold such rows in e4m3 codes under the power of two that their block's
largest value needs.
"""
from __future__ import annotations

import math
import random

import torch

own = False

E4M3 = torch.float8_e4m3fn
TOP = 448.0                    # the largest e4m3 number
MOST_FLOPS = 3.8e12            # a drawn case at most: the longest listed chunk's
MOST_SCORES = 8_600_000_000    # scores that the plain form holds at once, padded


def listed():
    return [
        # one user's next token: launch latency
        {"name": "attend one", "kind": "attend", "B": 1, "n": 1, "one": 0, "Hq": 32, "Hkv": 8, "D": 128, "G": 64, "page": 64, "L": 4096, "mix": 1},
        # a decoding batch in mid-flight, ragged contexts
        {"name": "attend batch", "kind": "attend", "B": 64, "n": 1, "one": 0, "Hq": 32, "Hkv": 8, "D": 128, "G": 64, "page": 256, "L": 8192, "mix": 2},
        # one long context without grouped heads, finer blocks
        {"name": "attend long", "kind": "attend", "B": 1, "n": 1, "one": 0, "Hq": 32, "Hkv": 32, "D": 128, "G": 32, "page": 128, "L": 65536, "mix": 3},
        # short turns on top of their conversations, narrow heads
        {"name": "attend turns", "kind": "attend", "B": 16, "n": 7, "one": 3, "Hq": 16, "Hkv": 4, "D": 64, "G": 32, "page": 64, "L": 3000, "mix": 4},
        # a serving step that decodes most sequences and takes in chunks of a few prompts
        {"name": "attend mixed", "kind": "attend", "B": 40, "n": 512, "one": 36, "Hq": 32, "Hkv": 8, "D": 128, "G": 64, "page": 256, "L": 8192, "mix": 5},
        # packed chunks of prompts with cached beginnings
        {"name": "attend chunks", "kind": "attend", "B": 10, "n": 1000, "one": 0, "Hq": 32, "Hkv": 8, "D": 128, "G": 32, "page": 64, "L": 16001, "mix": 6},
        # the last chunk of one long document
        {"name": "attend document", "kind": "attend", "B": 1, "n": 8192, "one": 0, "Hq": 32, "Hkv": 8, "D": 128, "G": 64, "page": 256, "L": 32768, "mix": 7},
        # one user's next token: launch latency
        {"name": "append one", "kind": "append", "fmt": "b8+", "B": 1, "n": 1, "one": 0, "Hq": 32, "Hkv": 8, "D": 128, "G": 64, "page": 64, "L": 4096, "rot": 128, "pairs": False, "places": False, "krot": False, "mix": 8},
        # a decoding batch's next tokens
        {"name": "append batch", "kind": "append", "fmt": "b8+", "B": 128, "n": 1, "one": 0, "Hq": 32, "Hkv": 8, "D": 128, "G": 32, "page": 64, "L": 2000, "rot": 128, "pairs": False, "places": False, "krot": False, "mix": 9},
        # drafted trees, whose rotation goes by the depth in the tree, partly rotated heads in pairs
        {"name": "append drafts", "kind": "append", "fmt": "f16+", "B": 24, "n": 16, "one": 5, "Hq": 16, "Hkv": 4, "D": 64, "G": 32, "page": 64, "L": 1500, "rot": 32, "pairs": True, "places": True, "krot": False, "mix": 10},
        # chunks of prompts with cached beginnings
        {"name": "append chunks", "kind": "append", "fmt": "b8+", "B": 10, "n": 1000, "one": 0, "Hq": 32, "Hkv": 8, "D": 128, "G": 64, "page": 64, "L": 6001, "rot": 128, "pairs": False, "places": False, "krot": False, "mix": 11},
        # a long prompt, whose rotated rows go on to its own attention
        {"name": "append prompt", "kind": "append", "fmt": "b8+", "B": 2, "n": 16384, "one": 0, "Hq": 32, "Hkv": 8, "D": 128, "G": 64, "page": 256, "L": 16384, "rot": 128, "pairs": False, "places": False, "krot": True, "mix": 12},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "append", "append"])
    while True:
        hkv = rng.choice([1, 2, 4, 8, 16])
        D = rng.choice([64, 128, 128])
        c = {"kind": kind, "B": _log(rng, 1, 96), "n": rng.choice([1, 1, _log(rng, 2, 40), _log(rng, 2, 8192)]), "one": 0, "Hq": hkv * rng.choice([1, 2, 4, 5, 7, 8, 16]),
             "Hkv": hkv, "D": D, "G": rng.choice([32, 64]), "page": rng.choice([64, 128, 256]), "mix": rng.randrange(1 << 20)}
        if c["n"] > 1 and rng.random() < 0.5:
            c["one"] = rng.randrange(c["B"])
        if kind == "attend":
            c["L"] = _log(rng, max(64, c["n"]), 131072)
            if c["L"] >= c["n"] and work(c)["flops"] <= MOST_FLOPS and c["B"] * c["Hq"] * c["n"] * c["L"] <= MOST_SCORES and c["B"] * c["L"] * hkv * D <= 1 << 30:
                return c
            continue
        c.update(fmt=rng.choice(["f16+", "b8+", "b8+"]), L=_log(rng, max(64, c["n"]), 16384), rot=D // rng.choice([1, 1, 2]), pairs=rng.random() < 0.4,
                 places=rng.random() < 0.3, krot=rng.random() < 0.4)
        if c["L"] >= c["n"] and sum(_new(c)) * (c["Hq"] + 2 * hkv) * D <= 1 << 27 and c["B"] * c["L"] * hkv * D <= 1 << 28:
            return c


# ------------------------------------------------------------------- sizes --
def _new(c):
    """New tokens of each sequence: one for the first `one`, spread over the logarithm for the others, the most among them."""
    r = random.Random(c["mix"] * 31 + 7)
    most = c["B"] - c["one"]
    new = [1] * c["one"] + [_log(r, max(1, c["n"] // 16), c["n"]) for _ in range(most)]
    new[-1] = c["n"]
    return new


def _lens(c):
    """Positions of each sequence with its new tokens: spread over the logarithm, the longest among them."""
    r, new = random.Random(c["mix"] * 1009 + c["B"]), _new(c)
    lens = [max(n, _log(r, max(1, c["L"] // 32), c["L"])) for n in new]
    lens[-1] = c["L"]
    return lens


def work(case):
    c, new = case, _new(case)
    T, D, Hq, Hkv = sum(new), c["D"], c["Hq"], c["Hkv"]
    if c["kind"] == "attend":
        lens = _lens(c)
        seen = sum(n * (x - n) + n * (n + 1) // 2 for x, n in zip(lens, new))
        return {"bytes": 2 * Hkv * sum(x * D + 2 * -(-x // c["G"]) for x in lens) + 4 * T * Hq * D, "flops": 4 * D * Hq * seen}
    row = D if c["fmt"] == "b8+" else 2 * D
    return {"bytes": T * (2 * D * (2 * Hq + 2 * Hkv + (Hkv if c["krot"] else 0)) + 2 * Hkv * row), "flops": 3 * T * (Hq + Hkv) * c["rot"]}


# ------------------------------------------------------------------ inputs --
def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class State:
    """What a program holds between steps."""


def _power(top):
    """The smallest power of two, from 2^-24 to 2^15, whose 448-fold is not below top >= 0 (fp32)."""
    m, e = torch.frexp(top)
    e = torch.where(m <= TOP / 512, e - 9, e - 8)
    return torch.ldexp(torch.ones_like(top), torch.where(top == 0, -24, e).clamp(-24, 15))


def _cache(c, pages, gen, size):
    """One tensor's page pool of N(0, size^2) rows and its scales."""
    x = torch.empty((pages, c["Hkv"], c["page"], c["D"]), dtype=torch.float16, device="cuda").normal_(0, size, generator=gen)
    if c.get("fmt") == "f16+":
        return x, None
    out, scales = torch.empty_like(x, dtype=E4M3), torch.empty((pages, c["Hkv"], c["page"] // c["G"]), dtype=torch.float16, device="cuda")
    for i in range(0, pages, 512):                        # in parts: fp32 copies of all would be large
        y = x[i:i + 512].float().unflatten(2, (-1, c["G"]))
        s = _power(y.abs().amax((-1, -2)))
        scales[i:i + 512] = s.half()
        out[i:i + 512] = (y / s[..., None, None]).flatten(2, 3).to(E4M3)
    return out, scales


def prepare(case, seed):
    c, s = dict(case), State()
    new, lens = _new(c), _lens(c)
    s.c, s.new, s.seq = c, new, lens
    gen = torch.Generator("cuda").manual_seed(int(seed))
    need = [-(-x // c["page"]) for x in lens]
    ids = list(range(sum(need) + 2))
    random.Random(seed).shuffle(ids)
    s.host = [[ids.pop() for _ in range(n)] for n in need]
    s.table = _int32([row + [-1] * (max(need) - len(row)) for row in s.host])
    s.cap = c["L"]
    T = sum(new)
    # one token each needs no bounds
    s.cu = None if T == c["B"] and max(new) == 1 else _int32([sum(new[:i]) for i in range(len(new) + 1)])
    s.lens = _int32(lens)
    # rows of a cache that grows are smaller than the new ones, so that held blocks are scaled anew
    size = 0.5 if c["kind"] == "append" else 1.0
    s.k, s.ks = _cache(c, sum(need) + 2, gen, size)
    s.v, s.vs = _cache(c, sum(need) + 2, gen, size)
    if c["kind"] == "attend":
        s.q = torch.empty((T, c["Hq"], c["D"]), dtype=torch.float16, device="cuda").normal_(generator=gen)
    else:
        qkv = torch.empty((T, c["Hq"] + 2 * c["Hkv"], c["D"]), dtype=torch.float16, device="cuda").normal_(generator=gen)
        s.q, s.kn, s.vn = qkv.split([c["Hq"], c["Hkv"], c["Hkv"]], 1)
        s.start = _int32([x - n for x, n in zip(lens, new)])
        s.freq = (10000.0 ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64) / c["rot"])).float().cuda()
        s.places = None
        if c["places"]:                                   # depths in a tree: no row further than its own position
            r = random.Random(seed + 1)
            s.places = _int32([x - n + r.randint(0, i) for x, n in zip(lens, new) for i in range(n)])
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------- plain forms --
def _bounds(s):
    """cu [B + 1] in 64 bits."""
    return torch.arange(s.c["B"] + 1, device="cuda") if s.cu is None else s.cu.long()


def _values(pool, scales, ids, G):
    """fp32 rows [B, Hkv, pages * page_rows, D] of the pages ids [B, pages]."""
    x = pool.view(torch.uint8)[ids].view(E4M3).float().unflatten(3, (-1, G))          # [B, pages, Hkv, blocks, G, D]
    return (x * scales[ids].float()[..., None, None]).flatten(3, 4).transpose(1, 2).flatten(2, 3)


def _attend(s):
    c = s.c
    B, Hq, Hkv, D, N = c["B"], c["Hq"], c["Hkv"], c["D"], max(s.new)
    cu, ids = _bounds(s), s.table.long().clamp(min=0)
    T = s.q.shape[0]
    at = torch.arange(N, device="cuda")
    q = s.q[(cu[:-1, None] + at).clamp_(max=T - 1)].float().transpose(1, 2).reshape(B * Hkv, Hq // Hkv * N, D)
    k = _values(s.k, s.ks, ids, c["G"]).reshape(B * Hkv, -1, D)
    cap = k.shape[1]
    x = (q @ k.transpose(1, 2).contiguous()).mul_(D ** -0.5).view(B, Hq, N, cap)
    del k
    last = (s.lens - (cu[1:] - cu[:-1]))[:, None] + at                                # [B, N]: the last position that a row sees
    x.masked_fill_((torch.arange(cap, device="cuda") > last[..., None])[:, None], -math.inf)
    x.sub_(x.amax(-1, keepdim=True)).exp_()
    x.div_(x.sum(-1, keepdim=True))
    o = x.view(B * Hkv, -1, cap) @ _values(s.v, s.vs, ids, c["G"]).reshape(B * Hkv, cap, D)
    o = o.view(B, Hq, N, D).half()
    tok = torch.arange(T, device="cuda")
    seq = torch.bucketize(tok, cu[1:], right=True)
    return o[seq, :, tok - cu[seq]]


def _rotate(x, turn, rot, pairs):
    """x [T, H, D] with its first rot dimensions turned, turn = (cos, sin) [T, 1, rot / 2]."""
    cos, sin = turn
    r = x[..., :rot]
    a, b = (r[..., 0::2], r[..., 1::2]) if pairs else r.chunk(2, -1)
    new = (a * cos - b * sin, a * sin + b * cos)
    new = torch.stack(new, -1).flatten(-2) if pairs else torch.cat(new, -1)
    return torch.cat([new, x[..., rot:]], -1)


def _write(s, pool, scales, x, page, row, seq):
    """The rows x [T, Hkv, D] (fp32) into the pool at (page, row) [T]."""
    c = s.c
    if scales is None:
        pool[page, :, row] = x.half()
        return
    G, per = c["G"], c["page"] // c["G"]
    flat = scales.transpose(1, 2).reshape(-1, c["Hkv"]).float()                        # [pages * per, Hkv]
    block = page * per + row // G
    first = s.start.long()                                                             # the block that a sequence begins in
    held = first % G
    lead = s.table.long().gather(1, (first // c["page"])[:, None])[:, 0].clamp(min=0) * per + first % c["page"] // G
    need = torch.zeros_like(flat).index_reduce_(0, block, x.abs().amax(-1), "amax")
    touched = torch.zeros(len(flat), dtype=torch.bool, device="cuda").index_fill_(0, block, True)
    kept = torch.zeros(len(flat), dtype=torch.bool, device="cuda").index_put_((lead,), held > 0)
    now = torch.where(touched[:, None], torch.maximum(_power(need), torch.where(kept[:, None], flat, 0.0)), flat)
    # what the sequences' first blocks hold, under the new scales
    codes = pool.view(torch.uint8)
    at = torch.arange(G, device="cuda")
    p, r = (lead // per)[:, None].expand(-1, G), (lead % per * G)[:, None] + at
    old = codes[p, :, r].view(E4M3).float() * (flat[lead] / now[lead])[:, None, :, None]       # [B, G, Hkv, D]
    stays = (at < held[:, None])[..., None, None]
    codes[p, :, r] = torch.where(stays, old.to(E4M3).view(torch.uint8), codes[p, :, r])
    codes[page, :, row] = (x / now[block][..., None]).to(E4M3).view(torch.uint8)
    scales.copy_(now.view(-1, per, c["Hkv"]).transpose(1, 2))


def _append(s):
    c, cu = s.c, _bounds(s)
    tok = torch.arange(s.q.shape[0], device="cuda")
    seq = torch.bucketize(tok, cu[1:], right=True)
    pos = s.start.long()[seq] + tok - cu[seq]
    angle = (pos if s.places is None else s.places).double()[:, None, None] * s.freq.double()
    turn = angle.cos().float(), angle.sin().float()
    q, k = (_rotate(x.float(), turn, c["rot"], c["pairs"]) for x in (s.q, s.kn))
    page, row = s.table.long()[seq, pos // c["page"]], pos % c["page"]
    _write(s, s.k, s.ks, k, page, row, seq)
    _write(s, s.v, s.vs, s.vn.float(), page, row, seq)
    return q.half(), k.half() if c["krot"] else None, s.k, s.v, s.ks, s.vs


# --------------------------------------------------------------------- run --
def run(s):
    c = s.c
    if not own:
        return _attend(s) if c["kind"] == "attend" else _append(s)
    import voltattn_amd.torch_ops  # noqa: F401  (registers torch.ops.voltattn)
    ops = torch.ops.voltattn
    if c["kind"] == "attend":
        return ops.attend_paged(s.q, s.k, s.v, s.ks, s.vs, s.table, s.cu, s.lens, "b8+", s.cap, c["G"])
    q, k = ops.append_rope(s.q, s.kn, s.vn, s.freq, s.cu, s.start, s.places, s.table, s.k, s.v, s.ks, s.vs, c["fmt"], c["G"], c["pairs"], c["krot"])
    return q, k if c["krot"] else None, s.k, s.v, s.ks, s.vs


# ------------------------------------------------------------------- exact --
def _exact_rows(s, pool, scales, b, h):
    """float64 rows of sequence b's head h."""
    pages = torch.tensor(s.host[b], device="cuda")
    code = pool[pages, h].double() if pool.dtype != E4M3 else pool.view(torch.uint8)[pages, h].view(E4M3).double()
    return (code * scales[pages, h].double().repeat_interleave(s.c["G"], 1)[..., None]).flatten(0, 1)


def _exact_attend(s):
    c, at = s.c, 0
    out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    g = c["Hq"] // c["Hkv"]
    for b, (n, x) in enumerate(zip(s.new, s.seq)):
        for h in range(c["Hkv"]):
            k, v = (_exact_rows(s, t, sc, b, h)[:x] for t, sc in ((s.k, s.ks), (s.v, s.vs)))
            for i in range(0, n, 4096):                   # blocks of queries
                e = min(n, i + 4096)
                for j in range(h * g, h * g + g):
                    w = s.q[at + i:at + e, j].double() @ k.T / math.sqrt(c["D"])
                    w += torch.full_like(w, -math.inf).triu(x - n + i + 1)
                    out[at + i:at + e, j] = torch.softmax(w, -1) @ v
        at += n
    return out


def _exact_append(s):
    c, at = s.c, 0
    # as complex numbers: a pair times e^(i angle)
    where = s.places.tolist() if s.places is not None else [x - n + i for x, n in zip(s.seq, s.new) for i in range(n)]
    phase = torch.outer(torch.tensor(where, dtype=torch.float64, device="cuda"), s.freq.double())
    phase = torch.polar(torch.ones_like(phase), phase)[:, None]

    def turned(x):
        x, R = x.double().clone(), c["rot"]
        a, b = (slice(0, R, 2), slice(1, R, 2)) if c["pairs"] else (slice(0, R // 2), slice(R // 2, R))
        z = torch.complex(x[..., a].contiguous(), x[..., b].contiguous()) * phase
        x[..., a], x[..., b] = z.real, z.imag
        return x

    q, k = turned(s.q), turned(s.kn)
    done = []
    for pool, scales, x in ((s.k, s.ks, k), (s.v, s.vs, s.vn.double())):
        out = pool.double()
        sc = None if scales is None else scales.double()
        row0 = 0
        for b, (n, end) in enumerate(zip(s.new, s.seq)):
            p = end - n
            while p < end:
                step = c["G"] if sc is not None else c["page"]
                stop = min(end, p // step * step + step)
                page, r = s.host[b][p // c["page"]], p % c["page"]
                new = x[row0:row0 + stop - p].transpose(0, 1)                          # [Hkv, rows, D]
                if sc is None:
                    out[page, :, r:r + stop - p] = new
                else:
                    i = r // step
                    need = torch.exp2(torch.ceil(torch.log2(new.abs().amax((1, 2)) / TOP))).clamp(2.0 ** -24, 2.0 ** 15)
                    if r % step:
                        need = torch.maximum(need, sc[page, :, i])
                        old = out[page, :, i * step:r] * (sc[page, :, i] / need)[:, None, None]
                        out[page, :, i * step:r] = old.float().to(E4M3).double()
                    sc[page, :, i] = need
                    out[page, :, r:r + stop - p] = (new / need[:, None, None]).float().to(E4M3).double()
                row0 += stop - p
                p = stop
        done.append((out, sc))
    return q, k if c["krot"] else None, done[0][0], done[1][0], done[0][1], done[1][1]


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_attend(s) if s.c["kind"] == "attend" else _exact_append(s)
