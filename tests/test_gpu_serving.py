"""GPU: the serving operators together, as a server uses them, on one page pool: pages for the
prompts (resize_pages), their rows appended (append_kv) and attended (prefill), single steps
(decode_paged), sequences forked (fork_pages), drafts verified (decode_tree), the accepted ones
moved together (compact_kv) and the rest given back (resize_pages). Every attention is checked in
64 bits against each sequence's own list of rows, quantized anew, and every page's holders
against the tables."""
import subprocess
from pathlib import Path

import pytest
import torch

import voltattn_amd.torch_ops  # noqa: F401
from tests import attn64

pytestmark = pytest.mark.gpu
ops = torch.ops.voltattn
BITS = {"f16+": 16, "q8+": 8, "q4+": 4, "q3+": 3}
HQ, HKV = 8, 2


def _int(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


class Server:
    def __init__(self, fmt, D, G, page, pages, wide):
        self.fmt, self.bits, self.D, self.G, self.page, self.wide = fmt, BITS[fmt], D, G, page, wide
        lead = (pages, HKV, page)
        if self.bits == 16:
            self.pools = [torch.zeros(lead + (D,), dtype=torch.float16, device="cuda") for _ in "kv"]
            self.scales = [None, None]
        else:
            self.pools = [torch.zeros(lead + (D * self.bits // 8,), dtype=torch.uint8, device="cuda")
                          for _ in "kv"]
            self.scales = [torch.zeros(lead + (D // G,), dtype=torch.float16, device="cuda") for _ in "kv"]
        self.refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
        self.table = torch.empty((0, wide), dtype=torch.int32, device="cuda")
        self.rows = []                                      # of every sequence: [(k, v)] of [HKV, D] fp16
        self.gen = torch.Generator("cuda").manual_seed(len(fmt) + D)

    def lens(self):
        return [len(r) for r in self.rows]

    def new(self, *lead):
        return torch.randn(lead + (self.D,), generator=self.gen, device="cuda").half()

    def resize(self, new):
        assert int(ops.resize_pages(self.table, self.refs, _int(self.lens()), _int(new), self.page)) == 0
        self.check_pages(new)

    def check_pages(self, lens):
        held = [self.table[b, :-(-n // self.page)] for b, n in enumerate(lens)]
        for b, h in enumerate(held):
            assert (h >= 0).all() and (self.table[b, len(h):] == -1).all()
        assert torch.equal(self.refs, torch.bincount(torch.cat(held), minlength=len(self.refs)).int())

    def append(self, b, k, v):
        """k, v [n, HKV, D] behind sequence b's rows."""
        start = _int([len(self.rows[b])])
        for x, pool, sc in zip((k, v), self.pools, self.scales):
            ops.append_kv(x.transpose(0, 1).contiguous()[None], start, self.table[b:b + 1], pool, sc, self.fmt, self.G)
        self.rows[b] += list(zip(k, v))

    def stored(self, b, h):
        """Sequence b's K and V rows of a head as its cache should hold them, and V's scales."""
        k, v = (torch.stack([r[i][h] for r in self.rows[b]]) for i in (0, 1))
        if self.bits == 16:
            return k, v, torch.ones_like(v)
        (k, ks), (v, vs) = (ops.quantize(x.float().contiguous(), self.bits, self.G) for x in (k, v))
        return ops.dequantize(k, ks, self.bits, self.G), ops.dequantize(v, vs, self.bits, self.G), vs.double().repeat_interleave(self.G, -1)

    def check(self, b, q, got, seen):
        """q and got [n, HQ, D]; seen [n, rows]."""
        for h in range(HKV):
            k, v, vs = self.stored(b, h)
            for i in range(h * HQ // HKV, (h + 1) * HQ // HKV):
                attn64.check(got[:, i], *attn64.attend(q[:, i], k, v, seen, vs), (self.fmt, b, i))

    def prompts(self, lens):
        self.rows = [[] for _ in lens]
        self.table = torch.full((len(lens), self.wide), -1, dtype=torch.int32, device="cuda")
        self.resize(lens)
        x = self.new(sum(lens), HQ + 2 * HKV)
        q, k, v = x.split([HQ, HKV, HKV], 1)                # slices of one projection
        cu = [sum(lens[:i]) for i in range(len(lens) + 1)]
        got = ops.prefill(q, k, v, _int(cu))
        for b, n in enumerate(lens):
            self.append(b, k[cu[b]:cu[b + 1]], v[cu[b]:cu[b + 1]])
            part = slice(cu[b], cu[b + 1])
            for i in range(HQ):                             # over the rows themselves, not the cache's
                h = i * HKV // HQ
                attn64.check(got[part, i], *attn64.attend(q[part, i], k[part, h], v[part, h], torch.ones((n, n), device="cuda").tril().bool()))

    def step(self):
        self.resize([n + 1 for n in self.lens()])
        for b in range(len(self.rows)):
            self.append(b, self.new(1, HKV), self.new(1, HKV))
        q = self.new(len(self.rows), HQ)
        got = ops.decode_paged(q, *self.pools, *self.scales, self.table, _int(self.lens()), self.fmt, self.wide * self.page, self.G)
        for b, n in enumerate(self.lens()):
            self.check(b, q[b:b + 1], got[b:b + 1], torch.ones((1, n), dtype=torch.bool, device="cuda"))

    def fork(self, parents):
        self.table, lens, missing = ops.fork_pages(self.table, _int(self.lens()), _int(parents), self.refs, *self.pools, *self.scales, self.fmt, self.G)
        assert int(missing) == 0
        self.rows = [list(self.rows[p]) for p in parents]
        assert lens.tolist() == self.lens()
        self.check_pages(self.lens())

    def verify(self, ups, sizes, keep):
        """ups: each draft's parent (-1: the context); keep: the accepted drafts of each sequence."""
        ctx, T = self.lens(), len(ups)
        self.resize([c + n for c, n in zip(ctx, sizes)])
        masks = []
        for i, up in enumerate(ups):
            masks.append(1 << i | (masks[up] if up >= 0 else 0))
        for b, n in enumerate(sizes):
            if n:
                self.append(b, self.new(n, HKV), self.new(n, HKV))
        q = self.new(len(ctx), T, HQ)
        got = ops.decode_tree(q, *self.pools, *self.scales, self.table, _int(ctx), _int(sizes), _int([masks] * len(ctx), torch.int64),
                              self.fmt, self.wide * self.page, self.G)
        for b, n in enumerate(sizes):
            assert (got[b, n:] == 0).all()
            if n:
                seen = [[True] * ctx[b] + [bool(masks[i] >> j & 1) for j in range(n)] for i in range(n)]
                self.check(b, q[b, :n], got[b, :n], torch.tensor(seen, device="cuda"))
        wide = [k + [0] * (T - len(k)) for k in keep]
        ops.compact_kv(*self.pools, *self.scales, self.table, _int(ctx), _int(wide), _int([len(k) for k in keep]), self.fmt, self.G)
        before = self.lens()
        self.rows = [r[:c] + [r[c + i] for i in k] for r, c, k in zip(self.rows, ctx, keep)]
        assert int(ops.resize_pages(self.table, self.refs, _int(before), _int(self.lens()), self.page)) == 0
        self.check_pages(self.lens())


@pytest.mark.parametrize("fmt", list(BITS))
@pytest.mark.parametrize("D,G,page", [(128, 32, 64), (64, 64, 128)])
def test_prompts_to_verified_drafts(fmt, D, G, page):
    s = Server(fmt, D, G, page, pages=40, wide=6)
    s.prompts([70, 1, 128, 190])
    s.step()
    s.step()
    s.fork([0, 2, 0, 1, 0])                                 # one sequence three times, one not at all
    s.step()
    ups = [-1, 0, 0, 1, 1, 2]
    s.verify(ups, [6, 3, 0, 1, 6], [[0, 2, 5], [0], [], [], [0, 1, 4]])
    s.step()
    s.fork([4, 4, 1])
    s.verify(ups, [6, 6, 6], [[0, 1, 3], [0], [0, 2]])
    s.step()
    assert int(ops.resize_pages(s.table, s.refs, _int(s.lens()), _int([0, 0, 0]), page)) == 0
    assert (s.refs == 0).all() and (s.table == -1).all()


def test_the_cpp_mirror_serves():
    """tests/cli's serving cases: the same operators through voltattn.hpp, against its single steps."""
    cli = Path(__file__).resolve().parent.parent / "build" / "voltattn"
    r = subprocess.run([str(cli), "--selftest-ex"], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-2000:]
    assert "all serving cases passed" in r.stdout and r.stdout.count("serve ") == 4
