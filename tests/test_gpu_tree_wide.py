"""GPU: the tree kernel's widest row blocks (128 query rows) in every format, row length and
group size, against float64 attention. They are taken where all rows of a K/V head are more than
64 and the batch has over four K/V tiles for each CU, so the batches here are that large, and
every case asserts the form that it runs in."""
import pytest
import torch

import voltattn_amd as va
import voltattn_amd.torch_ops  # noqa: F401
from tests.test_gpu_tree import Case, _int, ops

pytestmark = pytest.mark.gpu

CTX = [2100, 0, 1, 777, 2099, 64, 1500, 2047]
ROWS = [("f16+", 128, 32), ("f16+", 64, 32)] + [(f, D, G) for f in ("q8+", "q4+", "q3+") for D in (128, 64) for G in (32, 64)]


def _wide(fmt, D=128, G=32, ctx=CTX, T=33, group=4, Hkv=2, sizes=None, **kw):
    """A Case that the widest row blocks run, by the workspace that they ask for."""
    c = Case(fmt, ctx, T, Hkv * group, Hkv, D, G, sizes=sizes, **kw)
    shape = va.PagedShape(len(ctx), Hkv * group, Hkv, D, G, c.page, c.block_table.shape[1], c.pages, c.cap)
    f = {"f16+": va.Fmt.F16M, "q8+": va.Fmt.Q8M, "q4+": va.Fmt.Q4M, "q3+": va.Fmt.Q3M}[fmt]
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    per_cu = 3 if D == 128 or fmt == "f16+" else 4
    assert va.tree_ws_bytes(f, shape, T) == 2 * per_cu * cus * 128 * (D + 2) * 4, "not the widest row blocks"
    return c


@pytest.mark.parametrize("fmt,D,G", ROWS)
def test_ragged_contexts_and_trees(fmt, D, G):
    c = _wide(fmt, D, G, sizes=[33, 33, 7, 32, 0, 1, 33, 16], seed=D + G)
    c.check(c.run())


@pytest.mark.parametrize("fmt", ["f16+", "q4+"])
@pytest.mark.parametrize("T,group,page", [(64, 2, 64), (64, 8, 512), (17, 5, 128), (13, 10, 64)])
def test_rows_and_pages(fmt, T, group, page):
    c = _wide(fmt, ctx=[2100 + 7 * i for i in range(16)], T=T, group=group, page=page, chain=True, seed=T)
    c.check(c.run())


@pytest.mark.parametrize("fmt", ["f16+", "q8+", "q3+"])
def test_one_long_context_in_pieces(fmt):
    c = _wide(fmt, ctx=[33001], seed=1)
    got = c.run()
    c.check(got)
    assert torch.equal(c.run(), got)


@pytest.mark.parametrize("fmt", ["f16+", "q4+"])
def test_nothing_visible_is_zero(fmt):
    c = _wide(fmt, seed=2)
    c.masks[1] = [0] * 20 + [1 << i for i in range(20, 33)]
    got = c.run()
    assert (got[1, :20] == 0).all()
    c.check(got)


@pytest.mark.parametrize("fmt", ["f16+", "q8+"])
def test_bad_pages_and_lengths_reach_their_sequence_only(fmt):
    c = _wide(fmt, seed=3)
    want = c.run()
    others = [b for b in range(len(CTX)) if b != 3]
    for bad in (-1, c.pages, 1 << 30):
        t = c.block_table.clone()
        t[3, 5] = bad
        got = c.run(table=t)
        assert got[3].isnan().all() and torch.equal(got[others], want[others])
    for n in (-1, c.cap - 32, 1 << 30):
        got = c.run(ctx=_int(CTX[:3] + [n] + CTX[4:]))
        assert got[3].isnan().all()
        c.check(got, skip=(3,))


@pytest.mark.parametrize("fmt,D,G", ROWS)
def test_infinite_and_nan_values_reach_the_rows_that_see_them_only(fmt, D, G):
    """A draft's values (quantized: one group's scale), infinite or NaN: the drafts that do not see it are as
    without. A position of the context before the tiles with drafts: every draft has them."""
    c = _wide(fmt, D, G, seed=4 + D + G)
    want = c.run()
    b, ctx, at = 4, CTX[4], 16
    sees = torch.tensor([bool(m >> at & 1) for m in c.masks[b]], device="cuda")
    assert sees.any() and not sees.all()
    lo, hi = (8, 40) if c.bits == 16 else (0, G)
    others = [i for i in range(len(CTX)) if i != b]
    for kind in (float("inf"), -float("inf"), float("nan")):
        for j in (ctx + at, 100):
            page, row = c.table[b][j // c.page], j % c.page
            v = (c.v if c.bits == 16 else c.vs).clone()
            if c.bits == 16:
                v[page, 0, row, lo:hi] = kind
                got = c.run(v=v)
                code = torch.ones(hi - lo, device="cuda", dtype=torch.double)
            else:
                v[page, 0, row, 0] = kind
                got = c.run(vs=v)
                ones = torch.ones((1, 1, D // G), device="cuda", dtype=torch.half)
                code = ops.dequantize(c.v[page:page + 1, 0, row:row + 1].contiguous(), ones, c.bits, G)[0, 0, lo:hi].double()
            who = sees if j >= ctx else torch.ones_like(sees)
            assert torch.equal(got[others], want[others]) and torch.equal(got[b, ~who], want[b, ~who])
            assert torch.equal(got[b, :, 4:], want[b, :, 4:])           # the other K/V head
            x = got[b, who][:, :4]
            assert torch.equal(x[..., hi:], want[b, who][:, :4, hi:]) and torch.equal(x[..., :lo], want[b, who][:, :4, :lo])
            x = x[..., lo:hi].double()
            if j >= ctx:
                odd = (code * kind).expand_as(x)
                assert torch.equal(x.isnan(), odd.isnan()) and torch.equal(x > 65504, odd > 65504) and torch.equal(x < -65504, odd < -65504)
            else:
                assert not x.isfinite().any()


@pytest.mark.parametrize("fmt", ["f16+", "q4+"])
def test_other_stream_and_graph(fmt):
    c = _wide(fmt, seed=5)
    args = [_int(c.ctx), _int(c.sizes), c.mask()]

    def call():
        return ops.decode_tree(c.q, c.k, c.v, c.ks, c.vs, c.block_table, *args, fmt, c.cap, 32)

    want = call()
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
        args[0].copy_(_int([max(0, n - 10 * i) for n in c.ctx]))
        eager = call()
        out.fill_(7)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), i
