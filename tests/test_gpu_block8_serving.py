"""GPU: a serving loop on the block format: pages handed out (resize_pages), a projection's rows rotated
and written (append_rope), prompts attended as they are (prefill) and everything new from the cache
(attend_paged), step after step, as a captured step and on two streams at once."""
import pytest
import torch

import voltattn_amd.torch_ops  # noqa: F401
from tests import attn_bound, block8

pytestmark = pytest.mark.gpu
ops = torch.ops.voltattn
HQ, HKV, D, G, PAGE, PAGES, WIDE = 8, 2, 128, 32, 64, 40, 8


def _int(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Cache:
    def __init__(self, B, seed):
        self.B = B
        self.g = torch.Generator("cuda").manual_seed(seed)
        self.table = torch.full((B, WIDE), -1, dtype=torch.int32, device="cuda")
        self.refs = torch.zeros(PAGES, dtype=torch.int32, device="cuda")
        self.lens = [0] * B
        self.places = [[] for _ in range(B)]
        self.freq = (10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)).float().cuda()
        # what lies in pages that nothing has been written to: codes and scales of any value
        self.pools = [torch.randint(0, 256, (PAGES, HKV, PAGE, D), generator=self.g, device="cuda", dtype=torch.uint8).view(block8.E4M3) for _ in "kv"]
        self.scales = [torch.randn((PAGES, HKV, PAGE // G), generator=self.g, device="cuda").half() for _ in "kv"]

    def rows(self, T):
        size = float(torch.exp2(torch.randint(-3, 4, (1,), generator=self.g, device="cuda").float()))   # every step's rows another size
        x = (torch.randn((T, HQ + 2 * HKV, D), generator=self.g, device="cuda") * size).half()
        return x.split([HQ, HKV, HKV], 1)

    def grow(self, new):
        old, self.start = _int(self.lens), _int(self.lens)
        self.lens = [a + b for a, b in zip(self.lens, new)]
        assert int(ops.resize_pages(self.table, self.refs, old, _int(self.lens), PAGE)) == 0
        return _int([sum(new[:i]) for i in range(self.B + 1)])

    def write(self, x, cu, start):
        return ops.append_rope(*x, self.freq, cu, start, None, self.table, *self.pools, *self.scales, "b8+", G, False, True)

    def attend(self, q, cu, lens):
        return ops.attend_paged(q, *self.pools, *self.scales, self.table, cu, lens, "b8+", WIDE * PAGE, G)

    def check(self, got, q, new):
        """Every new row against attention in 64 bits over what the cache stands for."""
        k, v = (block8.values(p, s) for p, s in zip(self.pools, self.scales))
        at = 0
        for b, (n, t) in enumerate(zip(self.lens, new)):
            seen = torch.arange(n, device="cuda") <= (n - t + torch.arange(t, device="cuda"))[:, None]
            for i in range(HQ):
                kr, vr = (block8.rows(x, self.table[b], n, i * HKV // HQ) for x in (k, v))
                out, bound = attn_bound.attend(q[at:at + t, i], kr, vr, seen)
                off = (got[at:at + t, i].double() - out).abs()
                assert (off <= bound).all(), (b, i, float((off / bound).max()))
            at += t


STEPS = [[70, 1, 130], [1, 1, 1], [5, 1, 3], [1, 1, 1], [64, 33, 1], [1, 1, 1]]


def test_steps():
    c = Cache(3, 1)
    for s, new in enumerate(STEPS):
        places = torch.tensor([n + i for n, t in zip(c.lens, new) for i in range(t)], device="cuda")
        cu = c.grow(new)
        x = c.rows(sum(new))
        q, k = c.write(x, cu, c.start)
        for got, (want, off) in zip((q, k), (block8.rotate(y, places, c.freq, False) for y in x[:2])):
            assert ((got.double() - want).abs() <= off + 2.0 ** -11 * (want.abs() + off) + 2.0 ** -25).all()
        c.check(c.attend(q, cu, _int(c.lens)), q, new)
        # the cache's rows are the rows: half a step of e4m3 at the block's scale, which is below
        # 2 / 448 of the largest value that its rows of this step or the held ones have
        if s == 0:
            vals = [block8.values(p, z) for p, z in zip(c.pools, c.scales)]
            at = 0
            for b, t in enumerate(new):
                for vv, y in zip(vals, (k, x[2])):
                    for h in range(HKV):
                        held, want = block8.rows(vv, c.table[b], t, h), y[at:at + t, h].double()
                        scale = torch.cat([block8.need(want[i:i + G].abs().max()).expand(min(G, t - i)) for i in range(0, t, G)])[:, None]
                        # (k is the rotated row rounded to fp16: off by 2^-11 from what was quantized, which may
                        # move a value to the next code and a block's scale to the double)
                        assert ((held - want).abs() <= want.abs() * (2.0 ** -4 + 2.0 ** -10) + scale * 2.0 ** -9).all()
                at += t
            pre = ops.prefill(q, k, x[2].contiguous(), cu)
            at = 0
            for t in new:
                seen = torch.ones(t, t, dtype=torch.bool, device="cuda").tril()
                for i in range(HQ):
                    out, bound = attn_bound.attend(q[at:at + t, i], k[at:at + t, i * HKV // HQ].double(), x[2][at:at + t, i * HKV // HQ].double(), seen)
                    assert ((pre[at:at + t, i].double() - out).abs() <= bound).all()
                at += t
    assert int(ops.resize_pages(c.table, c.refs, _int(c.lens), _int([0] * 3), PAGE)) == 0 and (c.refs == 0).all()


def test_a_captured_step():
    """Tokens of every sequence: the graph's replays give what eager calls on the same cache give."""
    c = Cache(3, 2)
    for new in ([70, 1, 130], [1, 1, 1]):
        cu = c.grow(new)
        q, _ = c.write(c.rows(sum(new)), cu, c.start)
        c.attend(q, cu, _int(c.lens))
    c.lens = [n + 8 for n in c.lens]
    assert int(ops.resize_pages(c.table, c.refs, _int([n - 8 for n in c.lens]), _int(c.lens), PAGE)) == 0
    lens = _int([n - 8 for n in c.lens])
    x = torch.empty((3, HQ + 2 * HKV, D), dtype=torch.float16, device="cuda")

    def step():
        q, _ = c.write(x.split([HQ, HKV, HKV], 1), None, lens)
        lens.add_(1)
        return c.attend(q, None, lens)

    state = [*c.pools, *c.scales]
    before = [t.view(torch.uint8).clone() for t in state]
    first = lens.clone()
    x.normal_(generator=c.g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    got, inputs = [], []
    for t, z in zip(state, before):
        t.view(torch.uint8).copy_(z)
    lens.copy_(first)
    for i in range(6):
        x.normal_(generator=c.g)
        inputs.append(x.clone())
        graph.replay()
        got.append(out.clone())
        if i % 2:
            torch.cuda.synchronize()
            ops.attend_paged(torch.ones_like(out), *c.pools, *c.scales, c.table, None, lens, "b8+", WIDE * PAGE, G)   # eager work between
    after = [t.view(torch.uint8).clone() for t in state]
    for t, z in zip(state, before):
        t.view(torch.uint8).copy_(z)
    lens.copy_(first)
    for y, g in zip(inputs, got):
        x.copy_(y)
        assert torch.equal(step(), g)
    assert all(torch.equal(t.view(torch.uint8), z) for t, z in zip(state, after))


def test_two_streams_at_once():
    """Two caches, each on its own stream: the same as one after the other."""
    def run(seed, steps):
        c = Cache(3, seed)
        outs = []
        for new in steps:
            cu = c.grow(new)
            q, _ = c.write(c.rows(sum(new)), cu, c.start)
            outs.append(c.attend(q, cu, _int(c.lens)))
        return c, outs

    want = [run(s, STEPS)[1] for s in (3, 4)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    caches, outs = [], [[], []]
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            caches.append(Cache(3, 3 + i))
    for new in STEPS:
        work = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                work.append((caches[i].grow(new), caches[i].rows(sum(new))))
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                cu, x = work[i]
                q, _ = caches[i].write(x, cu, caches[i].start)
                outs[i].append(caches[i].attend(q, cu, _int(caches[i].lens)))
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        assert all(torch.equal(a, b) for a, b in zip(w, o))
