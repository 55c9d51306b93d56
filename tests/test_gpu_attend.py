"""GPU: attention over a cache in 8 bits with a scale for each block of positions and head
(va_attend_paged, torch.ops.voltattn.attend_paged) against float64 attention over the values
that the cache stands for (attn_bound's derived bound): one token and many, at the borders of
tiles (128 and 64 positions, 32 to a wave), row blocks (16, 32, 128 rows) and pages."""
import math

import pytest
import torch

import voltattn_amd.torch_ops  # noqa: F401
from tests import attn_bound, block8

pytestmark = pytest.mark.gpu
ops = torch.ops.voltattn


def _int(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Case:
    """Sequences with lens positions, the last new of them new, their pages scattered over a pool."""

    def __init__(self, lens, new, Hq=8, Hkv=2, D=128, G=64, page=64, seed=0, size=1.0):
        self.lens, self.new, self.Hq, self.Hkv, self.D, self.G, self.page = lens, new, Hq, Hkv, D, G, page
        g = torch.Generator("cuda").manual_seed(seed + 7)
        need = [-(-max(n, 0) // page) for n in lens]
        self.pages = sum(need) + 3
        perm = torch.randperm(self.pages, generator=g, device="cuda").tolist()
        self.host = [[perm.pop() for _ in range(n)] for n in need]
        wide = max(max(need), 1) + 1
        self.table = _int([r + [-1] * (wide - len(r)) for r in self.host])
        self.cap = wide * page
        self.cu = _int([sum(new[:i]) for i in range(len(new) + 1)])
        self.seq = _int(lens)
        draw = lambda *s: torch.randn(s, generator=g, device="cuda")          # noqa: E731
        # the sizes of blocks differ by powers of two, so that neighbours have different scales
        self.spread = lambda n: torch.exp2(torch.randint(-2, 3, (n, Hkv, page // G, 1, 1), generator=g, device="cuda").float())  # noqa: E731
        self.pools, self.scales = [], []
        for _ in "kv":
            x = (draw(self.pages, Hkv, page // G, G, D) * self.spread(self.pages) * size).flatten(2, 3)
            p, s = block8.pack(x, G)
            self.pools.append(p)
            self.scales.append(s)
        self.q = draw(sum(new), Hq, D).half()

    def run(self, cu="own", **kw):
        a = dict(q=self.q, table=self.table, cu=self.cu if cu == "own" else cu, seq=self.seq, cap=self.cap)
        a.update(kw)
        return ops.attend_paged(a["q"], *self.pools, *self.scales, a["table"], a["cu"], a["seq"], "b8+", a["cap"], self.G)

    def check(self, got, skip=(), what=""):
        k, v = (block8.values(p, s) for p, s in zip(self.pools, self.scales))
        g, at = self.Hq // self.Hkv, 0
        for b, (n, t) in enumerate(zip(self.lens, self.new)):
            if b not in skip:
                ctx = n - t
                blind = max(0, min(t, -ctx))                     # rows that see nothing
                assert (got[at:at + blind] == 0).all(), (what, b)
                seen = torch.arange(max(n, 0), device="cuda") <= (ctx + torch.arange(t, device="cuda"))[:, None]
                for h in range(self.Hkv if t > blind else 0):
                    kr, vr = (block8.rows(x, self.host[b], n, h) for x in (k, v))
                    for i in range(h * g, h * g + g):
                        out, bound = attn_bound.attend(self.q[at + blind:at + t, i], kr, vr, seen[blind:])
                        off = (got[at + blind:at + t, i].double() - out).abs()
                        assert (off <= bound).all(), (what, b, i, float((off / bound).max()))
            at += t


LENGTHS = [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 640, 1025]


@pytest.mark.parametrize("D,G", [(64, 32), (64, 64), (128, 32), (128, 64)])
@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (4, 4)])
def test_one_token(D, G, Hq, Hkv):
    c = Case(LENGTHS, [1] * len(LENGTHS), Hq, Hkv, D, G, seed=D + G)
    got = c.run(cu=None)
    c.check(got)
    assert torch.equal(got, c.run())                             # bounds of one row each: the same plan


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 8, 15, 16, 17, 31, 32, 33, 40, 64, 65, 127, 128, 129, 200])
@pytest.mark.parametrize("D,G", [(64, 32), (128, 64)])
def test_new_tokens(n, D, G):
    for Hq, Hkv in ((4, 1), (2, 2)):
        c = Case([n, n + 1, n + 63, n + 200, n + 700], [n] * 5, Hq, Hkv, D, G, seed=n)
        c.check(c.run(), what=(Hq, Hkv))


@pytest.mark.parametrize("D,G", [(64, 64), (128, 32), (128, 64)])
@pytest.mark.parametrize("lens,new", [([700, 800], [700, 520]), ([513], [512]), ([3000, 900], [257, 900]), ([1100, 70], [1090, 1])])
def test_long_chunks(D, G, lens, new):
    """Blocks of 256 rows, whole and in part."""
    c = Case(lens, new, 16, 2, D, G, 128, seed=sum(new))
    c.check(c.run())


@pytest.mark.parametrize("which", [0, 1])
def test_long_chunks_with_values_that_are_not_finite(which):
    """NaN codes, a page outside the pool and an infinite scale among the new rows of blocks of 256 rows."""
    c = Case([800], [700], 8, 1, 128, 32, 64, seed=20)
    want = c.run()
    sees = 100 + torch.arange(700, device="cuda")
    page = c.host[0][6]                                          # positions 384 .. 447
    c.pools[which].view(torch.uint8)[page, 0, 7, 9] = 0x7F
    got = c.run()
    bad = sees >= 391
    assert torch.equal(got[~bad], want[~bad])
    assert (got[bad][..., 9] if which else got[bad]).isnan().all()
    if which:
        got[..., 9] = want[..., 9]
        assert torch.equal(got, want)
    c.pools[which].view(torch.uint8)[page, 0, 7, 9] = 0
    want = c.run()
    c.scales[which][page, 0, 1] = math.inf
    got = c.run()
    bad = sees >= 416
    assert torch.equal(got[~bad], want[~bad]) and got[bad].isnan().all()
    c.scales[which][page, 0, 1] = 1.0
    table = c.table.clone()
    table[0, 9] = c.pages
    got = c.run(table=table)
    bad = sees >= 576
    assert got[bad].isnan().all() and got[~bad].isfinite().all()


@pytest.mark.parametrize("G", [32, 64])
@pytest.mark.parametrize("lens,new", [
    ([300, 5, 1000, 77, 1], [1, 5, 130, 0, 1]),                  # whole prompts, chunks, none, single tokens
    ([640] * 3 + [900], [1, 1, 1, 300]),
    ([0, 0, 40], [0, 0, 40]),
    ([100, 2000], [100, 33]),
])
def test_mixed_batches(lens, new, G):
    c = Case(lens, new, 8, 2, 128, G, 128, seed=sum(lens))
    c.check(c.run())


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (14, 2), (15, 3), (16, 1), (17, 1), (33, 1), (40, 8), (64, 1), (7, 7)])
@pytest.mark.parametrize("n", [1, 9])
def test_head_layouts(Hq, Hkv, n):
    c = Case([200, 333], [n, n], Hq, Hkv, 128, 32, seed=Hq)
    c.check(c.run())


@pytest.mark.parametrize("page", [64, 128, 1024])
@pytest.mark.parametrize("new", [[1, 1], [50, 3], [260, 1]])
def test_page_sizes(page, new):
    c = Case([1500, 700], new, 4, 2, 64, 64, page, seed=page)
    c.check(c.run())


@pytest.mark.parametrize("B", [64, 65, 150])
def test_many_sequences(B):
    """More than a wave plans at once."""
    lens = [(37 * i) % 211 + 1 for i in range(B)]
    c = Case(lens, [1] * B, 4, 2, 64, 32, seed=B)
    c.check(c.run(cu=None))
    new = [min(n, (5 * i) % 7) for i, n in enumerate(lens)]
    c = Case(lens, new, 4, 2, 64, 32, seed=B)
    c.check(c.run())


def test_long_context_in_pieces():
    """A context that every work-group has a piece of, several times 64 tiles each."""
    c = Case([70001], [1], 2, 1, 128, 64, 256, seed=1)
    c.check(c.run())
    c = Case([40000], [70], 4, 1, 64, 32, 256, seed=2)
    c.check(c.run())


def test_rows_that_see_nothing():
    """More new rows than positions: the first ones see nothing."""
    for new in ([5, 40, 3], [200, 140, 150]):
        c = Case([2, 33, 0], new, 4, 2, 128, 64, seed=3)
        c.check(c.run(), what=new)


def test_rows_of_no_sequence_are_zero():
    c = Case([100, 300], [40, 90], 4, 2, 128, 64, seed=4)
    q = torch.randn((400, 4, 128), device="cuda").half()
    cu = _int([70, 110, 200])
    got = c.run(q=q, cu=cu)
    assert (got[:70] == 0).all() and (got[200:] == 0).all()
    c.q = q[70:200]
    c.check(got[70:200])


def test_bounds_out_of_order_or_range():
    """A falling bound counts as its predecessor, one above the rows as their number, one below 0 as 0."""
    c = Case([200, 50, 150, 260], [100, 0, 150, 50], 2, 1, 64, 32, seed=5)
    c.check(c.run(cu=_int([-5, 100, 40, 250, 9999])))


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [70, 40, 100, 1]])
def test_lengths_out_of_range(new):
    c = Case([300, 200, 100, 50], new, 4, 2, 64, 64, seed=6)
    got = c.run(seq=_int([300, -1, 100, c.cap + 1]))
    c.check(got, skip=(1, 3))
    at = [sum(new[:i]) for i in range(5)]
    for b in (1, 3):
        assert got[at[b]:at[b + 1]].isnan().all()


@pytest.mark.parametrize("new", [[1, 1], [200, 150]])
@pytest.mark.parametrize("bad", [-1, 10 ** 6])
def test_pages_outside_the_pool(new, bad):
    """NaN for the rows that see the page's positions, and for no others."""
    c = Case([400, 390], new, 4, 2, 128, 32, 64, seed=7)
    table = c.table.clone()
    table[0, 4] = bad                                            # positions 256 .. 319
    got = c.run(table=table)
    c.check(got, skip=(0,))
    sees = (400 - new[0] + torch.arange(new[0], device="cuda")) >= 256
    assert got[:new[0]][sees].isnan().all()
    c.lens, c.new = [256], [int((~sees).sum())]
    if c.new[0]:
        c.check(got[:c.new[0]])


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("bits", [0x7C00, 0x7E00, 0xFC00])
@pytest.mark.parametrize("G", [32, 64])
def test_scales_that_are_not_finite(which, bits, G):
    for new in (1, 150):
        c = Case([300], [new], 4, 2, 128, G, 64, seed=8)
        c.scales[which].view(torch.int16)[c.host[0][3], 1, 1 if G == 32 else 0] = bits - 65536 if bits > 32767 else bits
        first = 224 if G == 32 else 192                          # the block's first position, of head 1
        got = c.run()
        sees = (300 - new + torch.arange(new, device="cuda")) >= first
        assert got[sees][:, 2:].isnan().all() and not got[:, :2].isnan().any() and not got[~sees].isnan().any()


@pytest.mark.parametrize("new", [1, 20, 150])
def test_nan_codes_reach_the_rows_that_see_them(new):
    c = Case([333], [new], 4, 2, 64, 32, 64, seed=9)
    p = 320                                                      # a position among the new ones if there are many
    page, row = c.host[0][p // 64], p % 64
    want = c.run()
    sees = (333 - new + torch.arange(new, device="cuda")) >= p
    for code in (0x7F, 0xFF):
        k0, v0 = (x.view(torch.uint8)[page, 0, row, 5].clone() for x in c.pools)
        c.pools[1].view(torch.uint8)[page, 0, row, 5] = code
        got = c.run()
        assert got[sees][:, :2, 5].isnan().all()
        got[:, :2, 5] = want[:, :2, 5]
        assert torch.equal(got, want)
        c.pools[1].view(torch.uint8)[page, 0, row, 5] = v0
        c.pools[0].view(torch.uint8)[page, 0, row, 5] = code
        got = c.run()
        assert got[sees][:, :2].isnan().all() and torch.equal(got[~sees], want[~sees]) and torch.equal(got[:, 2:], want[:, 2:])
        c.pools[0].view(torch.uint8)[page, 0, row, 5] = k0


def test_what_lies_behind_a_sequence_is_not_read():
    """NaN codes and scales behind the last position, and entries of the table there."""
    for new in (1, 40, 140):
        c = Case([170, 289], [new, new], 4, 2, 128, 32, 64, seed=10)
        want = c.run()
        for b, n in enumerate(c.lens):
            page, row = c.host[b][n // 64], n % 64
            for p, s in zip(c.pools, c.scales):
                p.view(torch.uint8)[page, :, row:] = 0x7F
                s[page, :, -(-row // 32):] = math.nan
        assert torch.equal(c.run(), want)
        c.check(want)


@pytest.mark.parametrize("new", [1, 12, 150])
@pytest.mark.parametrize("G", [32, 64])
def test_any_scales(new, G):
    """Scales that are no powers of two, subnormal, zero (its values are 0), negative (as positive), far apart."""
    c = Case([500], [new], 4, 2, 128, G, 64, seed=11)
    g = torch.Generator("cuda").manual_seed(1)
    for s in c.scales:
        s.copy_(torch.rand(s.shape, generator=g, device="cuda") * 0.03 + 0.001)
    page = c.host[0]
    c.scales[0][page[1], :, 0] = 0.0
    c.scales[1][page[2], :, 0] = 0.0
    c.scales[0][page[3], :, 0] *= -1
    c.scales[1][page[3], :, 0] *= -1
    c.scales[0][page[4], :, -1] = 3 * 2.0 ** -24
    c.check(c.run())
    c.scales[1][page[5], :, -1] = 37.5                           # values up to 16800 beside those of 1e-3
    c.scales[1][page[5], :, 0] = 5 * 2.0 ** -24
    c.check(c.run())


@pytest.mark.parametrize("e", [-24, -20, -9, 7, 15])
def test_all_scales_far_from_one(e):
    for new in (1, 140):
        c = Case([300], [new], 2, 1, 64, 32, 64, seed=12)
        c.scales[1].fill_(2.0 ** e)
        if e == 15:
            c.pools[1].view(torch.uint8).bitwise_and_(0x87)      # codes below 2^-6: the output fits fp16
        c.check(c.run())


@pytest.mark.parametrize("size", [0.0, 1e-3, 12.0])
@pytest.mark.parametrize("new", [1, 140])
def test_flat_and_peaked_scores(size, new):
    c = Case([700], [new], 4, 1, 128, 64, 64, seed=13)
    c.q = (c.q.float() * size).half()
    c.check(c.run())


@pytest.mark.parametrize("new", [1, 140])
def test_infinite_queries(new):
    """Rows whose scores are not finite are NaN; the others are as they were."""
    c = Case([300], [new], 4, 2, 64, 64, seed=14)
    want = c.run()
    c.q[new // 2, 1, 3] = math.inf
    got = c.run()
    assert not got[new // 2, 1].isfinite().any()
    got[new // 2, 1] = want[new // 2, 1]
    assert torch.equal(got, want)


def test_small_values_beside_large_ones():
    """Weights and values far below the largest keep their digits: a block of small values that has all the weight,
    beside one of large values that has next to none."""
    for new in (1, 140):
        c = Case([256], [new], 2, 1, 64, 32, 64, seed=15)
        page = c.host[0][1]
        c.scales[1][page, 0, 0] = 64.0                            # values up to 28672 ..
        k = c.pools[0].view(torch.uint8)
        far = block8.codes(torch.full((32, 64), -3.0, device="cuda", dtype=torch.float64), torch.tensor(2.0 ** -6, device="cuda"))
        k[page, 0, :32] = far                                     # .. at positions whose scores are far below the others
        c.scales[0][page, 0, 0] = 2.0 ** -6
        c.q = c.q.abs()
        c.check(c.run())


def test_repeated_calls_and_streams():
    """The same bits each time, and on two streams at once."""
    c = Case([3000, 17, 900], [1, 1, 1], 8, 2, 128, 64, seed=16)
    d = Case([900, 700], [300, 200], 8, 2, 128, 64, seed=17)
    want = c.run(), d.run()
    s = [torch.cuda.Stream() for _ in "ab"]
    torch.cuda.synchronize()
    got = []
    for i in range(6):
        with torch.cuda.stream(s[i % 2]):
            got.append((c if i // 2 % 2 else d).run())
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        assert torch.equal(x, want[0 if i // 2 % 2 else 1])


@pytest.mark.parametrize("lens,new", [([900, 77, 2000], [1, 1, 1]), ([900, 77, 2000], [300, 1, 140])])
def test_captured(lens, new):
    """Replays read lengths, tables and rows as they are then."""
    c = Case(lens, new, 8, 2, 128, 64, seed=18)
    c.run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = c.run()
    for shift in (0, 5, 64, 0):
        c.seq.copy_(_int([max(1, n - shift) for n in lens]))
        c.q.copy_(torch.randn_like(c.q, dtype=torch.float32).half())
        want = c.run()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_backward_raises_and_changes_are_noticed():
    c = Case([100], [3], 4, 2, 64, 32, seed=19)
    c.q.requires_grad_()
    out = c.run()
    with pytest.raises(RuntimeError, match="no gradient"):
        out.float().sum().backward()
    with torch.no_grad():
        assert not c.run().requires_grad
