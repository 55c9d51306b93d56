"""GPU: the rotating cache write (va_append_rope, torch.ops.voltattn.append_rope) against the
rotation in 64 bits (block8.rotate and its derived bound), the formats' own quantizer, and the
block format's rules."""
import math

import pytest
import torch

import voltattn_amd.torch_ops  # noqa: F401
from tests import block8

pytestmark = pytest.mark.gpu
ops = torch.ops.voltattn
BITS = {"f16": 16, "f16+": 16, "q8": 8, "q8+": 8, "q4": 4, "q4+": 4, "q3+": 3}


def _int(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _freq(rot, base=10000.0):
    return (base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)).float().cuda()


class Case:
    def __init__(self, fmt, start, new, Hq=4, Hkv=2, D=128, G=64, page=64, rot=None, seed=0, size=1.0, held=1.0, extra=0):
        self.fmt, self.start, self.new, self.Hq, self.Hkv, self.D, self.G, self.page = fmt, start, new, Hq, Hkv, D, G, page
        g = torch.Generator("cuda").manual_seed(seed + 3)
        need = [-(-max(s + n, 1) // page) for s, n in zip(start, new)]
        self.pages = sum(need) + 3
        perm = torch.randperm(self.pages, generator=g, device="cuda").tolist()
        self.host = [[perm.pop() for _ in range(n)] for n in need]
        wide = max(need) + extra
        self.table = _int([r + [-1] * (wide - len(r)) for r in self.host])
        self.cu = _int([sum(new[:i]) for i in range(len(new) + 1)])
        T = sum(new)
        self.qkv = (torch.randn((T, Hq + 2 * Hkv, D), generator=g, device="cuda") * size).half()
        self.q, self.k, self.v = self.qkv.split([Hq, Hkv, Hkv], 1)
        self.freq = _freq(rot or D)
        self.places = torch.tensor([s + i for s, n in zip(start, new) for i in range(n)], dtype=torch.int64, device="cuda")
        lead = (self.pages, Hkv, page)
        if fmt == "b8+":
            x = torch.randn(lead + (D,), generator=g, device="cuda") * held
            self.pools, self.scales = map(list, zip(*(block8.pack(x + i, G) for i in range(2))))
        elif BITS[fmt] == 16:
            self.pools, self.scales = [torch.zeros(lead + (D,), dtype=torch.float16, device="cuda") for _ in "kv"], [None, None]
        else:
            self.pools = [torch.zeros(lead + (D * BITS[fmt] // 8,), dtype=torch.uint8, device="cuda") for _ in "kv"]
            self.scales = [torch.zeros(lead + (D // G,), dtype=torch.float16, device="cuda") for _ in "kv"]

    def run(self, **kw):
        kw.setdefault("start", None)
        if kw["start"] is None:
            kw["start"] = _int(self.start)
        a = dict(q=self.q, k=self.k, v=self.v, freq=self.freq, cu=self.cu, positions=None, table=self.table,
                 pools=self.pools, scales=self.scales, interleaved=False, rotated_k=True, scaling=1.0)
        a.update(kw)
        return ops.append_rope(a["q"], a["k"], a["v"], a["freq"], a["cu"], a["start"], a["positions"], a["table"], *a["pools"], *a["scales"],
                               self.fmt, self.G, a["interleaved"], a["rotated_k"], a["scaling"])

    def places_of(self, i=0):
        return self.places

    def slots(self):
        """(row, page, row of the page) of every row that is written."""
        at = 0
        for b, (s, n) in enumerate(zip(self.start, self.new)):
            for i in range(n):
                p = s + i
                if 0 <= p < self.table.shape[1] * self.page:
                    page = int(self.table[b, p // self.page])
                    if 0 <= page < self.pages:
                        yield at + i, page, p % self.page
            at += n


def _near(got, want, off, what=""):
    """fp16 rows: the rotation's own error and one rounding, at most half a step (2^-11 of it, or 2^-25)."""
    bound = off + 2.0 ** -11 * (want.abs() + off) + 2.0 ** -25
    d = (got.double() - want).abs()
    assert (d <= bound).all(), (what, float((d / bound).max()))


def _check_rows(c, got, places=None, interleaved=False, scaling=1.0):
    places = c.places if places is None else places
    q, k = got
    _near(q, *block8.rotate(c.q, places, c.freq, interleaved, scaling), "q")
    if k.shape[0]:
        _near(k, *block8.rotate(c.k, places, c.freq, interleaved, scaling), "k")


def _check_blocks(c, before, places=None, interleaved=False, scaling=1.0):
    """The pools of the block format after a call, and that nothing else changed."""
    places = c.places if places is None else places
    k, off = block8.rotate(c.k, places, c.freq, interleaved, scaling)
    v = c.v.double()
    blocks = {}
    for r, page, row in c.slots():
        blocks.setdefault((page, row // c.G), []).append((r, row))
    for i, (x, d) in enumerate(((k, off), (v, torch.zeros_like(v)))):
        pool, scales = before[0][i].view(torch.uint8).clone(), before[1][i].clone()
        got, gs = c.pools[i].view(torch.uint8), c.scales[i]
        for (page, blk), rs in blocks.items():
            rows, at = [r for r, _ in rs], [w for _, w in rs]
            y, e = x[rows].transpose(0, 1), d[rows].transpose(0, 1)                    # [Hkv, rows, D]
            fin = torch.where(y.isfinite(), y.abs(), torch.zeros_like(y))
            top = fin.amax((1, 2))
            lo, hi = block8.need((fin - e).amax((1, 2)).clamp(min=0)), block8.need((fin + e).amax((1, 2)))
            assert torch.equal(lo, hi), "a border of the scale's rule: other inputs are wanted"
            first = min(at)
            held = first % c.G
            old = scales[page, :, blk].double()
            new = torch.maximum(hi, old) if held else hi
            assert torch.equal(gs[page, :, blk].double(), new), (i, page, blk, top)
            if held:
                keep = block8.codes(pool[page, :, blk * c.G:first].contiguous().view(block8.E4M3).double() * (old / new)[:, None, None], torch.ones((), device="cuda", dtype=torch.float64))
                pool[page, :, blk * c.G:first] = torch.where((old == new)[:, None, None], pool[page, :, blk * c.G:first], keep)
            scales[page, :, blk] = new.half()
            s = new[:, None, None]
            low, high = (block8.codes(z, s).view(block8.E4M3).double() for z in (y - e, y + e))
            code = got[page][:, at]
            z = code.contiguous().view(block8.E4M3).double()
            ok = (z >= low) & (z <= high) | (low.isnan() & z.isnan())
            assert ok.all(), (i, page, blk)
            pool[page][:, at] = code
        same = pool.view(block8.E4M3).double(), got.view(block8.E4M3).double()
        assert torch.equal(torch.nan_to_num(same[0], nan=1e9), torch.nan_to_num(same[1], nan=1e9)), i
        assert torch.equal(scales, gs), i


def _copy(c):
    return [p.clone() for p in c.pools], [None if s is None else s.clone() for s in c.scales]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,G", [(64, 32), (64, 64), (128, 32), (128, 64)])
@pytest.mark.parametrize("start,new", [
    ([0, 1, 31, 63, 64, 100], [1] * 6),                          # single tokens, blocks begun and held
    ([0, 5, 60, 64, 0, 7], [3, 70, 9, 64, 0, 1]),                # few rows over several blocks, none
    ([0, 17, 64, 130], [200, 100, 64, 33]),                      # many rows
])
def test_blocks(start, new, D, G, interleaved):
    c = Case("b8+", start, new, 4, 2, D, G, seed=D + G + len(new))
    before = _copy(c)
    got = c.run(interleaved=interleaved)
    _check_rows(c, got, interleaved=interleaved)
    _check_blocks(c, before, interleaved=interleaved)


@pytest.mark.parametrize("new", [[1, 1], [40, 2], [150, 90]])
def test_blocks_that_hold_rows(new):
    """New rows larger than the held ones scale them anew, smaller ones do not."""
    for held in (2.0 ** -6, 8.0):
        c = Case("b8+", [70, 33], new, 4, 2, 128, 64, 128, held=held, seed=int(held))
        before = _copy(c)
        c.run()
        _check_blocks(c, before)
        if held < 1:
            assert all(not torch.equal(a, b) for a, b in zip(before[1], c.scales))


def test_token_by_token_is_a_prompt():
    """Rows appended one by one leave the scales of a prompt, and its codes where no held code fell below e4m3's normal numbers."""
    c = Case("b8+", [0], [150], 4, 2, 64, 32, seed=5)
    d = Case("b8+", [0], [150], 4, 2, 64, 32, seed=5)
    c.run()
    for i in range(150):
        ops.append_rope(d.q[i:i + 1], d.k[i:i + 1], d.v[i:i + 1], d.freq, None, _int([i]), None, d.table, *d.pools, *d.scales, "b8+", 32)
    for h in d.host[0]:
        for a, b, s in zip(c.pools, d.pools, zip(c.scales, d.scales)):
            assert torch.equal(s[0][h], s[1][h])
            x, y = a[h].double(), b[h].double()
            near = (x - y).abs() <= 2.0 ** -9                    # a step of the subnormal numbers
            assert near.all() and torch.equal(x[x.abs() >= 2.0 ** -6], y[x.abs() >= 2.0 ** -6])


@pytest.mark.parametrize("fmt", list(BITS))
@pytest.mark.parametrize("D,G", [(64, 32), (128, 64)])
@pytest.mark.parametrize("start,new", [([0, 63, 100], [1, 1, 1]), ([3, 0, 64], [70, 1, 129])])
def test_row_formats_without_rotation(fmt, D, G, start, new):
    """Frequencies of 0: what append_kv writes of the same rows, bit for bit, pages of any size."""
    c = Case(fmt, start, new, 4, 2, D, G, 48 if len(set(new)) > 1 else 64, seed=D)
    c.freq = torch.zeros_like(c.freq)
    q, k = c.run()
    assert torch.equal(q, c.q) and torch.equal(k, c.k)
    for i, x in enumerate((c.k, c.v)):
        pool, sc = torch.zeros_like(c.pools[i]), None if c.scales[i] is None else torch.zeros_like(c.scales[i])
        at = 0
        for b, n in enumerate(new):
            ops.append_kv(x[at:at + n].transpose(0, 1).contiguous()[None], _int([start[b]]), c.table[b:b + 1], pool, sc, fmt, G)
            at += n
        assert torch.equal(pool, c.pools[i])
        assert sc is None or torch.equal(sc, c.scales[i])


@pytest.mark.parametrize("fmt", ["f16+", "q8+", "q4+", "q3+"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_row_formats_rotated(fmt, interleaved):
    """Stored k against the rotated rows: half a step of the codes (fp16: one rounding)."""
    c = Case(fmt, [5, 60], [90, 1], 6, 2, 128, 32, seed=21)
    got = c.run(interleaved=interleaved)
    _check_rows(c, got, interleaved=interleaved)
    want, off = block8.rotate(c.k, c.places, c.freq, interleaved)
    bits = BITS[fmt]
    for r, page, row in c.slots():
        if bits == 16:
            assert torch.equal(c.pools[0][page, :, row], got[1][r])
            assert torch.equal(c.pools[1][page, :, row], c.v[r])
            continue
        x = ops.dequantize(c.pools[0][page, :, row].contiguous(), c.scales[0][page, :, row].contiguous(), bits, 32).double()
        s = c.scales[0][page, :, row].double().repeat_interleave(32, -1)
        lim = {8: 127, 4: 7, 3: 3}[bits]
        # half a step, and what the largest value loses where its fp16 scale was rounded down (2^-11 of it)
        assert ((x - want[r]).abs() <= 0.5 * s + lim * s * 2.0 ** -11 + off[r] + 2.0 ** -20 * s).all()


@pytest.mark.parametrize("rot", [16, 32, 48, 64, 96, 112, 128])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("fmt", ["f16+", "b8+"])
def test_partly_rotated_heads(rot, interleaved, fmt):
    for new in ([1, 1], [40, 30]):
        c = Case(fmt, [3, 130], new, 3, 1, 128, 32, rot=rot, seed=rot)
        before = _copy(c)
        got = c.run(interleaved=interleaved)
        _check_rows(c, got, interleaved=interleaved)
        assert torch.equal(got[0][..., rot:], c.q[..., rot:]) and torch.equal(got[1][..., rot:], c.k[..., rot:])
        if fmt == "b8+":
            _check_blocks(c, before, interleaved=interleaved)


def test_rotation_by_given_positions_and_scaling():
    for fmt in ("b8+", "f16+"):
        for new in ([7, 1, 12], [60, 50, 40]):
            c = Case(fmt, [100, 0, 77], new, 4, 2, 64, 32, seed=8)
            g = torch.Generator("cuda").manual_seed(1)
            places = torch.randint(-500, 100000, (sum(new),), generator=g, device="cuda")
            before = _copy(c)
            got = c.run(positions=places.int(), scaling=1.375)
            _check_rows(c, got, places, scaling=1.375)
            if fmt == "b8+":
                _check_blocks(c, before, places, scaling=1.375)


def test_far_positions():
    """Angles of positions near 2^31 and their negatives: the rotation goes by them in 64 bits. (In 64 bits the reference's own
    angle is off by 2^-53 of up to 2^31 radians, the kernel's by three times that: 2^-20 together.)"""
    c = Case("f16+", [0], [8], 4, 2, 128, 64, seed=9)
    places = torch.tensor([2 ** 31 - 1, 2 ** 31 - 2, -2 ** 31, 2 ** 30 + 7, 123456789, 2 ** 24 + 1, 2 ** 24 + 3, 16777215], device="cuda")
    got = c.run(positions=places.int())
    want, off = block8.rotate(c.q, places, c.freq, False)
    _near(got[0], want, 3 * off)


@pytest.mark.parametrize("fmt", ["f16+", "q8+", "b8+"])
def test_rows_that_are_not_written(fmt):
    """Before position 0, past the table, on pages outside the pool: q and k are rotated all the same, the others written."""
    for new in ([10, 9, 6], [80, 100, 70]):
        c = Case(fmt, [-3, 120, 0], new, 4, 2, 64, 32, 64, seed=10, extra=1)
        c.table[2, 0] = -7
        c.table[1, 2 if new[1] < 20 else 3] = c.pages
        if fmt != "b8+":
            c.run()
            written = {(p, r) for _, p, r in c.slots()}
            for x in c.pools:
                for page in range(c.pages):
                    for row in range(c.page):
                        assert bool(x[page, :, row].any()) == ((page, row) in written), (page, row)
        else:
            before = _copy(c)
            got = c.run()
            _check_rows(c, got)
            _check_blocks(c, before)


def test_rows_of_no_sequence():
    for fmt in ("b8+", "q8+"):
        for T, cu in ((12, [2, 5, 5, 9]), (300, [20, 150, 100, 280])):
            new = [b - a for a, b in zip(cu, cu[1:])] if T == 12 else [130, 0, 130]
            c = Case(fmt, [4, 0, 60], new, 4, 2, 64, 32, seed=11)
            qkv = torch.randn((T, 8, 64), device="cuda").half()
            q, k, v = qkv.split([4, 2, 2], 1)
            got = c.run(q=q, k=k, v=v, cu=_int(cu))
            rest = torch.ones(T, dtype=torch.bool, device="cuda")
            rest[cu[0]:cu[-1]] = False
            assert (got[0][rest] == 0).all() and (got[1][rest] == 0).all()
            c.q, c.k, c.v = q[~rest], k[~rest], v[~rest]
            _check_rows(c, (got[0][~rest], got[1][~rest]))


def test_values_that_are_not_finite():
    """In the block format they become NaN and leave the block's scale to the others."""
    for new in ([1], [60], [150]):
        c = Case("b8+", [0], new, 4, 2, 64, 32, seed=12)
        c.v[0, 0, 3], c.v[0, 1, 9], c.v[-1, 0, 0] = math.inf, -math.inf, math.nan
        c.k[0, 1, 40], c.k[0, 1, 8] = math.nan, math.inf
        before = _copy(c)
        c.run()
        x = c.pools[1].view(torch.uint8)[c.host[0][0], :, 0].contiguous().view(block8.E4M3).float()
        assert x[0, 3].isnan() and x[1, 9].isnan() and int(x.isnan().sum()) == (3 if new == [1] else 2)
        c.k[0, 1, 40], c.k[0, 1, 8] = 0.0, 0.0                   # their pairs are NaN too: k by its scale alone
        y = c.pools[0].view(torch.uint8)[c.host[0][0], 1, 0].contiguous().view(block8.E4M3).float()
        assert y[[8, 40]].isnan().all() and int(y.isnan().sum()) == 2
        assert c.scales[0].isfinite().all() and c.scales[1].isfinite().all()
        del before


def test_extreme_sizes():
    """All zeros, the smallest numbers, the largest ones with a scaling that passes what the scale can hold."""
    for new in ([1], [40], [100]):
        for size, scaling in ((0.0, 1.0), (2.0 ** -24, 1.0), (2.0 ** -20, 2.0 ** -30), (60000.0, 1.0), (60000.0, 4096.0)):
            c = Case("b8+", [0], new, 2, 1, 64, 32, seed=13, size=1.0)
            x = torch.randn((new[0], 4, 64), device="cuda").clamp(-1, 1) * size
            q, k, v = x.half().split([2, 1, 1], 1)
            c.q, c.k, c.v = q, k, v
            before = _copy(c)
            c.run(scaling=scaling)
            _check_blocks(c, before, scaling=scaling)


@pytest.mark.parametrize("fmt", ["f16+", "b8+"])
def test_strides(fmt):
    for new in ([1, 1], [30, 40]):
        c = Case(fmt, [4, 90], new, 6, 3, 64, 32, seed=14)
        d = Case(fmt, [4, 90], new, 6, 3, 64, 32, seed=14)
        got = c.run()
        hm = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (d.q, d.k, d.v)]
        also = d.run(q=hm[0], k=hm[1], v=hm[2])
        for a, b in zip(got + tuple(c.pools), also + tuple(d.pools)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        e = Case(fmt, [4, 90], new, 6, 3, 64, 32, seed=14)       # one K/V head for three
        k1, v1 = e.k[:, :1].expand(-1, 3, -1), e.v[:, :1].expand(-1, 3, -1)
        _, k = e.run(k=k1, v=v1)
        assert torch.equal(k[:, 0], got[1][:, 0]) and torch.equal(k[:, 2], got[1][:, 0])


def test_many_sequences():
    for fmt in ("b8+", "q4+"):
        new = [(3 * i) % 5 for i in range(150)]
        c = Case(fmt, [(7 * i) % 90 for i in range(150)], new, 4, 2, 64, 32, seed=15)
        before = _copy(c)
        _check_rows(c, c.run())
        if fmt == "b8+":
            _check_blocks(c, before)
    c = Case("b8+", [(7 * i) % 90 for i in range(70)], [(40 * i) % 130 for i in range(70)], 2, 1, 64, 32, seed=16)
    before = _copy(c)
    _check_rows(c, c.run())
    _check_blocks(c, before)


def test_without_bounds_and_without_k():
    c = Case("b8+", [3, 64, 127], [1, 1, 1], 4, 2, 128, 64, seed=17)
    d = Case("b8+", [3, 64, 127], [1, 1, 1], 4, 2, 128, 64, seed=17)
    q, k = c.run()
    q2, k2 = d.run(cu=None, rotated_k=False)
    assert k2.shape == (0, 2, 128) and torch.equal(q, q2)
    for a, b in zip(c.pools, d.pools):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_captured():
    """Replays read starts, tables and rows as they are then."""
    c = Case("b8+", [5, 64, 100], [1, 40, 2], 4, 2, 128, 64, seed=18)
    d = Case("b8+", [5, 64, 100], [1, 40, 2], 4, 2, 128, 64, seed=18)
    start = _int(c.start)
    c.run(start=start)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = c.run(start=start)
    d.run()
    for shift in (0, 1, -5, 3):
        start.copy_(_int([s + shift for s in d.start]))
        c.qkv.copy_(torch.randn_like(c.qkv, dtype=torch.float32).half())
        d.qkv.copy_(c.qkv)
        want = d.run(start=start)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        for a, b in zip(c.pools + c.scales, d.pools + d.scales):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_backward_raises_and_changes_are_noticed():
    c = Case("f16+", [0], [3], 2, 1, 64, 32, seed=19)
    x = torch.ones_like(c.pools[0]).requires_grad_()
    y = (x * c.pools[0]).sum()
    c.run()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    q = c.q.detach().clone().requires_grad_()
    out, _ = c.run(q=q)
    with pytest.raises(RuntimeError, match="gradient|autograd"):
        out.float().sum().backward()
