"""GPU: attention of drafted tokens over a paged cache (va_decode_tree,
torch.ops.voltattn.decode_tree) against float64 attention of every sequence, draft and
head, in every tiled format, over the row blocks (32, 64, 128 query rows) and tiles (64 or
128 positions), ragged contexts and trees, and the cases whose outputs are defined to be
zero or NaN."""
import pytest
import torch

import voltattn_amd.torch_ops  # noqa: F401
from tests import attn64

pytestmark = pytest.mark.gpu
ops = torch.ops.voltattn
BITS = {"f16+": 16, "q8+": 8, "q4+": 4, "q3+": 3}


def _int(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


def _signed(m):
    return m - (1 << 64) if m >> 63 else m


class Case:
    """A pool with the sequences' pages scattered over it, the other rows full of random bytes (NaN
    patterns among them), and random trees."""

    def __init__(self, fmt, ctx, T, Hq, Hkv, D=128, G=32, page=64, sizes=None, seed=0, chain=False, vmag=1.0):
        g = torch.Generator("cuda").manual_seed(seed)
        self.fmt, self.bits, self.G, self.D, self.T, self.ctx = fmt, BITS[fmt], G, D, T, ctx
        self.Hq, self.Hkv, self.page = Hq, Hkv, page
        B = len(ctx)
        self.sizes = sizes or [T] * B
        need = [-(-(n + T) // page) for n in ctx]
        self.pages = sum(need) + 3
        ids = torch.randperm(self.pages, generator=torch.Generator().manual_seed(seed)).tolist()
        self.table = [[ids.pop() for _ in range(n)] for n in need]
        wide = max(need) + 1
        self.block_table = _int([r + [-1] * (wide - len(r)) for r in self.table])
        self.cap = max(ctx) + T
        lead = (self.pages, Hkv, page)
        x = [torch.randn(lead + (D,), generator=g, device="cuda") * m for m in (1.0, vmag)]
        if self.bits == 16:
            self.k, self.v, self.ks, self.vs = x[0].half(), x[1].half(), None, None
        else:
            (self.k, self.ks), (self.v, self.vs) = (ops.quantize(t, self.bits, G) for t in x)
        for b, row in enumerate(self.table):                # behind the sequence's last row: anything
            n = ctx[b] + self.sizes[b]
            for i, p in enumerate(row):
                r = max(0, min(page, n - i * page))
                for t in (self.k, self.v, self.ks, self.vs):
                    if t is not None:
                        t[p, :, r:].view(torch.uint8).fill_(255)
        self.q = torch.randn((B, T, Hq, D), generator=g, device="cuda").half()
        r = torch.Generator().manual_seed(seed + 1)
        self.masks = []
        for _ in range(B):
            m = []
            for i in range(T):
                up = i - 1 if chain else int(torch.randint(-1, max(i, 1), (1,), generator=r)) if i else -1
                m.append((1 << i) | (m[up] if up >= 0 else 0))
            self.masks.append(m)

    def mask(self):
        return _int([[_signed(m) for m in row] for row in self.masks], torch.int64)

    def run(self, **kw):
        a = dict(q=self.q, k=self.k, v=self.v, ks=self.ks, vs=self.vs, table=self.block_table, ctx=_int(self.ctx),
                 sizes=_int(self.sizes), mask=self.mask(), cap=self.cap)
        a.update(kw)
        return ops.decode_tree(a["q"], a["k"], a["v"], a["ks"], a["vs"], a["table"], a["ctx"], a["sizes"], a["mask"], self.fmt,
                               a["cap"], self.G)

    def _rows(self, pool, sc, b, h):
        x = torch.cat([pool[p, h] for p in self.table[b]])[:self.ctx[b] + self.sizes[b]]
        if self.bits == 16:
            return x, torch.ones_like(x)
        s = torch.cat([sc[p, h] for p in self.table[b]])[:x.shape[0]]
        return (ops.dequantize(x.contiguous(), s.contiguous(), self.bits, self.G), s.double().repeat_interleave(self.G, -1))

    def check(self, got, skip=()):
        g = self.Hq // self.Hkv
        # over 64 query rows to a K/V head the kernel rounds dequantized V values to fp16
        rounded = self.bits != 16 and self.T * g > 64
        for b in range(len(self.ctx)):
            n, c = self.sizes[b], self.ctx[b]
            if b in skip:
                continue
            assert (got[b, n:] == 0).all(), b
            seen = torch.tensor([[True] * c + [bool(m >> j & 1) for j in range(n)] for m in self.masks[b][:n]],
                                dtype=torch.bool, device="cuda").view(n, c + n)
            for h in range(self.Hkv if n else 0):
                k, _ = self._rows(self.k, self.ks, b, h)
                v, sv = self._rows(self.v, self.vs, b, h)
                for i in range(h * g, h * g + g):
                    attn64.check(got[b, :n, i], *attn64.attend(self.q[b, :n, i], k, v, seen, sv, rounded), (b, i))


@pytest.mark.parametrize("fmt", list(BITS))
@pytest.mark.parametrize("D,G", [(128, 32), (128, 64), (64, 32), (64, 64)])
@pytest.mark.parametrize("T,Hq,Hkv", [(1, 4, 2), (5, 8, 2), (16, 8, 2), (13, 10, 2), (64, 6, 2)])
def test_formats_and_row_blocks(fmt, D, G, T, Hq, Hkv):
    c = Case(fmt, [300, 1, 64, 127, 0], T, Hq, Hkv, D, G, seed=T + D)
    c.check(c.run())


@pytest.mark.parametrize("page", [64, 128, 512])
@pytest.mark.parametrize("ctx", [0, 1, 31, 32, 33, 63, 64, 65, 112, 127, 128, 129, 191, 255, 1000])
def test_context_lengths(ctx, page):
    for fmt, T, group in (("q8+", 16, 1), ("f16+", 16, 4), ("q4+", 33, 4)):
        c = Case(fmt, [ctx], T, 2 * group, 2, page=page, seed=ctx + page)
        c.check(c.run())


@pytest.mark.parametrize("fmt", list(BITS))
def test_long_context_in_pieces(fmt):
    c = Case(fmt, [9001], 8, 4, 1, seed=2)
    c.check(c.run())


@pytest.mark.parametrize("T,group", [(4, 4), (16, 4), (32, 8)])
def test_ragged_batch(T, group):
    ctx = [(977 * i) % 2100 for i in range(70)]              # more sequences than a wave scans at once
    sizes = [(5 * i) % (T + 1) for i in range(70)]
    c = Case("q8+", ctx, T, group, 1, D=64, sizes=sizes, seed=3, page=128)
    c.check(c.run())


def test_chain_and_no_sizes():
    c = Case("q8+", [100, 700], 40, 8, 2, chain=True, seed=4)
    c.check(c.run())
    assert torch.equal(c.run(), c.run(sizes=None))


def test_single_token_is_a_decode_step():
    c = Case("q8+", [99, 640, 5], 1, 8, 2, seed=5)
    want = ops.decode_paged(c.q[:, 0], c.k, c.v, c.ks, c.vs, c.block_table, _int([n + 1 for n in c.ctx]), "q8+", c.cap, 32)
    got = c.run()[:, 0]
    off = (got.double() - want.double()).abs()
    assert (off <= 2.0 ** -10 * (want.double().abs() + 1)).all()     # two fp16 results and the weights' rounding


@pytest.mark.parametrize("fmt", ["f16+", "q4+"])
def test_nothing_visible_is_zero(fmt):
    c = Case(fmt, [0, 0, 130], 12, 4, 2, seed=6, sizes=[12, 0, 7])
    c.masks = [[0] * 6 + [1 << i for i in range(6, 12)], [0] * 12, [0] * 12]
    got = c.run()
    assert (got[0, :6] == 0).all() and (got[1] == 0).all()
    c.check(got)


def test_bits_beyond_the_drafts_are_ignored():
    c = Case("q8+", [77], 9, 4, 2, sizes=[5], seed=7)
    want = c.run()
    c.masks = [[m | ~((1 << 5) - 1) & ((1 << 64) - 1) for m in row] for row in c.masks]
    assert torch.equal(c.run(), want)


@pytest.mark.parametrize("fmt", ["f16+", "q8+"])
def test_bad_page_reaches_its_sequence_only(fmt):
    c = Case(fmt, [300, 200, 500], 8, 4, 2, seed=8)
    want = c.run()
    for bad in (-1, c.pages, 1 << 30):
        t = c.block_table.clone()
        t[1, 2] = bad
        got = c.run(table=t)
        assert got[1].isnan().all()
        assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
    t = c.block_table.clone()
    t[1, -1] = 1 << 20                                      # behind its last position: not read
    assert torch.equal(c.run(table=t), want)


def test_lengths_out_of_range_give_nan():
    c = Case("q8+", [300, 200, 500, 100], 8, 4, 2, seed=9)
    want = c.run()
    for ctx, sizes in (([-1] + c.ctx[1:], c.sizes), ([c.cap - 7] + c.ctx[1:], c.sizes), ([1 << 30] + c.ctx[1:], c.sizes),
                       ([2 ** 31 - 1] + c.ctx[1:], c.sizes), (c.ctx, [9, 8, 8, 8]), (c.ctx, [-1, 8, 8, 8])):
        got = c.run(ctx=_int(ctx), sizes=_int(sizes))
        assert got[0].isnan().all()
        c.check(got, skip=(0,))
    assert torch.equal(c.run(), want)


def test_values_of_large_and_small_magnitude():
    for vmag in (2e-5, 1.0, 9000.0):
        for fmt in ("f16+", "q8+", "q4+", "q3+"):
            c = Case(fmt, [260], 8, 4, 2, vmag=vmag, seed=10)
            c.check(c.run())


def test_peaked_scores():
    c = Case("q8+", [700], 16, 4, 2, seed=11)
    c.q.mul_(20)
    c.check(c.run())


def test_other_stream_graph_and_repeat():
    c = Case("q8+", [300, 900, 40], 16, 8, 2, seed=12)
    args = [_int(c.ctx), _int(c.sizes), c.mask()]

    def call():
        return ops.decode_tree(c.q, c.k, c.v, c.ks, c.vs, c.block_table, *args, "q8+", c.cap, 32)

    want = call()
    assert torch.equal(call(), want)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = call()
    st.synchronize()
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    for i in range(3):
        c.q.normal_()
        args[0].copy_(_int([n - 10 * i for n in c.ctx]))
        eager = call()
        out.fill_(7)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), i


@pytest.mark.parametrize("fmt", list(BITS))
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,group", [(5, 4), (12, 4), (33, 4)])
def test_infinite_and_nan_drafts_reach_the_rows_that_see_them_only(fmt, D, T, group):
    """A draft whose values (quantized: one group's scale) are infinite or NaN: the drafts that do not see
    it are as without, those that do get the values' kind in its columns. The whole context is one piece,
    and many."""
    for ctx in (0, 100, 5000):
        c = Case(fmt, [ctx], T, 2 * group, 2, D, seed=T + ctx)
        want = c.run()
        c.sizes[0] = T
        at = T // 2
        page, row = c.table[0][(ctx + at) // c.page], (ctx + at) % c.page
        sees = torch.tensor([bool(m >> at & 1) for m in c.masks[0]], device="cuda")
        for kind in (float("inf"), -float("inf"), float("nan")):
            v = (c.v if c.bits == 16 else c.vs).clone()
            if c.bits == 16:
                v[page, 0, row, 8:40] = kind
                got = c.run(v=v)
                lo, sign = 8, torch.ones(32, device="cuda", dtype=torch.double)
            else:
                lo, x = 32, c.v[page:page + 1, 0, row:row + 1]
                ones = torch.ones((1, 1, D // 32), device="cuda", dtype=torch.half)
                sign = ops.dequantize(x.contiguous(), ones, c.bits, 32)[0, 0, 32:64].double()      # the codes: 0 times inf is NaN
                v[page, 0, row, 1] = kind
                got = c.run(vs=v)
            assert torch.equal(got[0, ~sees], want[0, ~sees]) and torch.equal(got[0, :, group:], want[0, :, group:])
            odd = (sign * kind).expand(int(sees.sum()), group, 32)
            x = got[0, sees][:, :group, lo:lo + 32].double()
            assert torch.equal(x.isnan(), odd.isnan()) and torch.equal(x > 65504, odd > 65504) and torch.equal(x < -65504, odd < -65504)
            rest = [i for i in range(D) if not lo <= i < lo + 32]
            assert torch.equal(got[0, sees][..., rest], want[0, sees][..., rest])
