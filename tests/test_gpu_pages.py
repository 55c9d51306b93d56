"""GPU: the page pool's operators (va_compact_kv, va_fork_pages, va_resize_pages and their
torch ops) against a model of the pool that does one thing after the other in plain Python.
Everything is whole numbers or copied bytes: equal or wrong."""
import random

import pytest
import torch

import voltattn_amd.torch_ops  # noqa: F401

pytestmark = pytest.mark.gpu
ops = torch.ops.voltattn
BITS = {"f16+": 16, "q8+": 8, "q4+": 4, "q3+": 3}


def _int(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _pools(fmt, pages, Hkv, page, D, G, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    out = []
    for _ in "kv":
        row = D * BITS[fmt] // 8
        x = torch.randint(0, 256, (pages, Hkv, page, row), generator=g, device="cuda", dtype=torch.uint8)
        s = None
        if BITS[fmt] == 16:
            x = x.view(torch.float16)
        else:
            s = torch.randint(0, 256, (pages, Hkv, page, 2 * D // G), generator=g, device="cuda", dtype=torch.uint8).view(torch.float16)
        out += [(x, s)]
    (k, ks), (v, vs) = out
    return k, v, ks, vs


def _bytes(t):
    return None if t is None else t.view(torch.uint8).clone()


def _same(pools, want):
    for t, w in zip(pools, want):
        if w is not None:
            assert torch.equal(t.view(torch.uint8), w)


class Pool:
    """The pool's bookkeeping, one page at a time."""

    def __init__(self, table, refs, page):
        self.table, self.refs, self.page = [list(r) for r in table], list(refs), page
        self.wide = len(self.table[0])

    def held(self, n):
        return -(-max(0, min(n, self.wide * self.page)) // self.page)

    def good(self, i):
        return 0 <= i < len(self.refs)

    def take(self):
        for i, r in enumerate(self.refs):
            if r == 0:
                self.refs[i] = 1
                return i
        return -1

    def resize(self, old, new):
        for row, a, b in zip(self.table, old, new):
            for i in range(self.held(b), self.held(a)):
                if self.good(row[i]):
                    self.refs[row[i]] -= 1
                row[i] = -1
        missing = 0
        for row, a, b in zip(self.table, old, new):
            for i in range(self.held(a), self.held(b)):
                row[i] = self.take()
                missing += row[i] < 0
        return missing

    def fork(self, lens, parents):
        """Returns (table, lens, missing, copies): copies = (from page, to page, rows)."""
        lens = [max(0, min(n, self.wide * self.page)) for n in lens]
        parents = [p if 0 <= p < len(lens) else -1 for p in parents]
        for p, n in enumerate(lens):
            kids = parents.count(p)
            for i in range(self.held(n)):
                if self.good(self.table[p][i]):
                    self.refs[self.table[p][i]] += (kids if i < n // self.page else min(kids, 1)) - 1
        table, new_lens, missing, copies = [], [], 0, []
        for c, p in enumerate(parents):
            n = lens[p] if p >= 0 else 0
            row = self.table[p][:self.held(n)] if p >= 0 else []
            row += [-1] * (self.wide - len(row))
            if n % self.page and p in parents[:c] and self.good(row[n // self.page]):
                src = row[n // self.page]
                row[n // self.page] = to = self.take()
                missing += to < 0
                if to >= 0:
                    copies.append((src, to, n % self.page))
            table.append(row)
            new_lens.append(n)
        return table, new_lens, missing, copies


def _fresh(rng, B, page, wide, spare, longest=None):
    """Tables of B sequences with pages of their own; some free pages among them."""
    lens = [rng.randrange(0, (longest or wide * page) + 1) for _ in range(B)]
    need = [-(-n // page) for n in lens]
    ids = list(range(sum(need) + spare))
    rng.shuffle(ids)
    table = [[ids.pop() for _ in range(n)] + [-1] * (wide - n) for n in need]
    refs = [1] * (sum(need) + spare)
    for i in ids:
        refs[i] = 0
    return table, refs, lens


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("B,page,wide", [(1, 64, 4), (7, 64, 9), (33, 16, 12), (140, 64, 5), (1100, 1, 6), (3, 7, 20000)])
def test_resize(seed, B, page, wide):
    rng = random.Random(seed * 1000 + B)
    table, refs, lens = _fresh(rng, B, page, wide, spare=(0, 3, 50, B, 5 * B, 9000)[seed], longest=min(wide, 60) * page)
    m = Pool(table, refs, page)
    t, r = _int(table), _int(refs)
    for step in range(4):
        new = [rng.choice([0, n, min(wide, 80) * page, rng.randrange(0, min(wide, 70) * page + 1)]) for n in lens]
        missing = m.resize(lens, new)
        got = ops.resize_pages(t, r, _int(lens), _int(new), page)
        assert int(got) == missing
        assert r.tolist() == m.refs
        assert t.tolist() == m.table
        lens = new


def test_resize_lengths_out_of_range():
    m = Pool([[0, 1, -1], [2, -1, -1]], [1, 1, 1, 0, 0, 0], 4)
    t, r = _int(m.table), _int(m.refs)
    old, new = [8, 4], [-3, 2 ** 31 - 1]
    assert int(ops.resize_pages(t, r, _int(old), _int(new), 4)) == m.resize(old, new)
    assert t.tolist() == m.table == [[-1, -1, -1], [2, 0, 1]] and r.tolist() == m.refs


def test_resize_ids_outside_the_pool():
    m = Pool([[9, -1, 0], [-7, 1, 2 ** 31 - 1]], [1, 1, 0], 4)
    t, r = _int(m.table), _int(m.refs)
    assert int(ops.resize_pages(t, r, _int([12, 12]), _int([0, 0]), 4)) == m.resize([12, 12], [0, 0])
    assert t.tolist() == m.table and r.tolist() == m.refs == [0, 0, 0]


def test_resize_scans_a_large_pool():
    """Free pages far apart in a pool of many scan rounds."""
    n, page = 70000, 64
    refs = [1] * n
    for i in range(0, n, 777):
        refs[i] = 0
    m = Pool([[-1] * 40 for _ in range(3)], refs, page)
    t, r = _int(m.table), _int(refs)
    new = [40 * page, 0, 39 * page]
    assert int(ops.resize_pages(t, r, _int([0, 0, 0]), _int(new), page)) == m.resize([0, 0, 0], new) == 0
    assert t.tolist() == m.table and r.tolist() == m.refs


@pytest.mark.parametrize("fmt", list(BITS))
@pytest.mark.parametrize("D,G", [(128, 32), (64, 64)])
@pytest.mark.parametrize("B,page,wide", [(1, 64, 3), (6, 64, 5), (5, 5, 9), (150, 64, 4)])
def test_fork(fmt, D, G, B, page, wide):
    rng = random.Random(B * 100 + D)
    table, refs, lens = _fresh(rng, B, page, wide, spare=3 * B + 4)
    k, v, ks, vs = _pools(fmt, len(refs), 2, page, D, G)
    pools = (k, v, ks, vs)
    m = Pool(table, refs, page)
    t, r = _int(table), _int(refs)
    for step, children in enumerate((B, B + 3, max(1, B // 2), 2 * B)):
        parents = [rng.randrange(-1, len(lens) + 1) if step == 1 else rng.randrange(len(lens)) for _ in range(children)]
        want = [_bytes(x) for x in pools]
        new_table, new_lens, missing, copies = m.fork(lens, parents)
        for src, dst, n in copies:
            for w in want:
                if w is not None:
                    w[dst, :, :n] = w[src, :, :n]
        t, got_lens, got_missing = ops.fork_pages(t, _int(lens), _int(parents), r, k, v, ks, vs, fmt, G)
        assert int(got_missing) == missing
        assert got_lens.tolist() == new_lens
        assert r.tolist() == m.refs
        assert t.tolist() == new_table
        _same(pools, want)
        m.table, lens = new_table, new_lens


def test_fork_without_free_pages():
    """Children whose copy finds no page hold -1 there; the others get theirs in order."""
    m = Pool([[0, 1], [2, 3]], [1, 1, 1, 1, 0], 64)
    k, v, ks, vs = _pools("q8+", 5, 1, 64, 64, 32)
    t, r = _int(m.table), _int(m.refs)
    parents = [0, 0, 0, 1, 1]
    table, lens, missing, _ = m.fork([100, 100], parents)
    t, got, miss = ops.fork_pages(t, _int([100, 100]), _int(parents), r, k, v, ks, vs, "q8+", 32)
    assert int(miss) == missing == 2 and t.tolist() == table and r.tolist() == m.refs and got.tolist() == lens


def test_fork_ids_outside_the_pool_and_odd_lengths():
    m = Pool([[0, 99], [1, 2], [3, -1]], [1, 1, 1, 1, 0, 0, 0], 64)
    k, v, ks, vs = _pools("f16+", 7, 1, 64, 64, 32)
    want = [_bytes(x) for x in (k, v, ks, vs)]
    lens, parents = [100, 2 ** 31 - 1, -5], [0, 0, 1, 1, 2, 2, 7, -1, 2 ** 31 - 1]
    table, new_lens, missing, copies = m.fork(lens, parents)
    assert not copies
    t, r = _int([[0, 99], [1, 2], [3, -1]]), _int([1, 1, 1, 1, 0, 0, 0])
    t, got, miss = ops.fork_pages(t, _int(lens), _int(parents), r, k, v, ks, vs, "f16+", 32)
    assert t.tolist() == table and got.tolist() == new_lens and int(miss) == missing and r.tolist() == m.refs
    _same((k, v, ks, vs), want)


def test_fork_many_children():
    """More children than the planning work-group has threads."""
    page, lens = 4, [6] * 30
    m = Pool([[2 * i, 2 * i + 1, -1] for i in range(30)], [1] * 60 + [0] * 2600, page)
    k, v, ks, vs = _pools("q4+", 2660, 1, page, 64, 64)
    t, r = _int(m.table), _int(m.refs)
    parents = [i % 30 for i in range(2500)]
    want = [_bytes(x) for x in (k, v, ks, vs)]
    table, new_lens, missing, copies = m.fork(lens, parents)
    for src, dst, n in copies:
        for w in want:
            w[dst, :, :n] = w[src, :, :n]
    t, got, miss = ops.fork_pages(t, _int(lens), _int(parents), r, k, v, ks, vs, "q4+", 64)
    assert t.tolist() == table and r.tolist() == m.refs and int(miss) == missing == 0
    _same((k, v, ks, vs), want)


def _compacted(pools, table, base, keep, counts, page):
    out = [_bytes(x) for x in pools]
    place = lambda b, p: (table[b][p // page], p % page) if 0 <= p < len(table[b]) * page and 0 <= table[b][p // page] < pools[0].shape[0] else None  # noqa: E731
    for b, (at, ks, n) in enumerate(zip(base, keep, counts)):
        for i, j in enumerate(ks[:max(0, min(n, len(ks)))]):
            src = place(b, at + j) if at >= 0 and j >= 0 else None
            dst = place(b, at + i) if at >= 0 else None
            if src and dst:
                for x, w in zip(pools, out):
                    if w is not None:
                        w[dst[0], :, dst[1]] = x.view(torch.uint8)[src[0], :, src[1]]
    return out


@pytest.mark.parametrize("fmt", list(BITS))
@pytest.mark.parametrize("D,G", [(128, 32), (64, 32), (128, 64), (64, 64)])
@pytest.mark.parametrize("n", [1, 7, 64])
def test_compact(fmt, D, G, n):
    rng = random.Random(n + D)
    for page in (64, 16, 5):
        B, wide = 9, -(-330 // page)
        ids = list(range(B * wide + 2))
        rng.shuffle(ids)
        table = [[ids.pop() for _ in range(wide)] for _ in range(B)]
        pools = _pools(fmt, B * wide + 2, 3, page, D, G)
        base = [rng.randrange(0, 200) for _ in range(B)]
        keep = [sorted(rng.sample(range(n), rng.randint(1, n))) for _ in range(B)]
        keep[0] = [rng.randrange(100) for _ in range(n)]                    # any order, repetitions
        counts = [len(x) for x in keep]
        counts[1], counts[2] = 0, -4
        keep = [x + [0] * (n - len(x)) for x in keep]
        want = _compacted(pools, table, base, keep, counts, page)
        ops.compact_kv(*pools, _int(table), _int(base), _int(keep), _int(counts), fmt, G)
        _same(pools, want)


def test_compact_out_of_range():
    """Rows from or to places outside the table or the pool are not written; counts above n are n."""
    table = [[3, 9, 1], [0, 2, -1], [4, 5, 6]]
    pools = _pools("q8+", 7, 2, 64, 128, 32)
    base, counts = [60, 126, -1], [99, 4, 4]
    keep = [[1, 5, 70, 80], [1, 2, -1, 10 ** 9], [0, 1, 2, 3]]
    want = _compacted(pools, table, base, keep, counts, 64)
    ops.compact_kv(*pools, _int(table), _int(base), _int(keep), _int(counts), "q8+", 32)
    _same(pools, want)


def test_compact_pools_of_small_alignment():
    """Quantized pools need 4-byte alignment only, scales 2."""
    D, G, page, Hkv = 128, 32, 64, 2
    raw = torch.randint(0, 256, (2, 4 * Hkv * page * D + 4), device="cuda", dtype=torch.uint8)
    sraw = torch.randint(0, 256, (2, 4 * Hkv * page * 8 + 2), device="cuda", dtype=torch.uint8)
    k, v = (raw[i, 4:].view(4, Hkv, page, D) for i in range(2))
    ks, vs = (sraw[i, 2:].view(torch.float16).view(4, Hkv, page, 4) for i in range(2))
    pools, table = (k, v, ks, vs), [[1, 2], [3, 0]]
    base, keep, counts = [50, 10], [[3, 9, 40], [1, 2, 60]], [3, 3]
    want = _compacted(pools, table, base, keep, counts, page)
    ops.compact_kv(*pools, _int(table), _int(base), _int(keep), _int(counts), "q8+", G)
    _same(pools, want)
    m = Pool([[1, 2], [3, -1]], [0, 1, 1, 1], page)
    want = [_bytes(x) for x in pools]
    _, _, _, copies = m.fork([100, 20], [0, 0])
    for src, dst, n in copies:
        for w in want:
            w[dst, :, :n] = w[src, :, :n]
    r = _int([0, 1, 1, 1])
    ops.fork_pages(_int([[1, 2], [3, -1]]), _int([100, 20]), _int([0, 0]), r, k, v, ks, vs, "q8+", G)
    assert r.tolist() == m.refs and copies
    _same(pools, want)


def test_graphs_replay_on_the_state_as_it_is():
    page = 64
    m = Pool([[0, 1, -1, -1], [2, -1, -1, -1]], [1, 1, 1] + [0] * 20, page)
    t, r = _int(m.table), _int(m.refs)
    old, new = _int([100, 30]), _int([200, 64])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        missing = ops.resize_pages(t, r, old, new, page)
    lens = [[100, 30], [200, 64], [10, 250], [0, 250]]
    for a, b in zip(lens, lens[1:]):
        old.copy_(_int(a))
        new.copy_(_int(b))
        g.replay()
        torch.cuda.synchronize()
        assert int(missing) == m.resize(a, b)
        assert t.tolist() == m.table and r.tolist() == m.refs


def test_fork_graph_replays():
    page, fmt = 64, "q8+"
    m = Pool([[0, 1, -1], [2, 3, -1]], [1, 1, 1, 1] + [0] * 12, page)
    k, v, ks, vs = pools = _pools(fmt, 16, 2, page, 128, 32)
    t, r, lens, par = _int(m.table), _int(m.refs), _int([100, 70]), _int([0, 0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        nt, nl, miss = ops.fork_pages(t, lens, par, r, k, v, ks, vs, fmt, 32)
        t.copy_(nt)
        lens.copy_(nl)
    n = [100, 70]
    for parents in ([0, 0], [1, 0], [1, 1]):
        par.copy_(_int(parents))
        want = [_bytes(x) for x in pools]
        table, n, missing, copies = m.fork(n, parents)
        for src, dst, rows in copies:
            for w in want:
                w[dst, :, :rows] = w[src, :, :rows]
        g.replay()
        torch.cuda.synchronize()
        m.table = table
        assert t.tolist() == table and r.tolist() == m.refs and lens.tolist() == n and int(miss) == missing
        _same(pools, want)
