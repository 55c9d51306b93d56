"""GPU: causal attention of packed prompts (va_prefill, torch.ops.voltattn.prefill) against
float64 attention of every sequence and head, at the tile borders (128 query rows, 64 K/V
rows, 32-row waves), over strided and shared heads, gaps around and between the sequences,
and values that must not reach other rows."""
import pytest
import torch

import voltattn_amd as va
import voltattn_amd.torch_ops  # noqa: F401
from tests import attn64

pytestmark = pytest.mark.gpu
ops = torch.ops.voltattn


def _inputs(n, Hq, Hkv, D, seed, scale=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return tuple(torch.randn((n, h, D), generator=g, device="cuda").mul_(s).half() for h, s in ((Hq, scale), (Hkv, 1.0), (Hkv, 1.0)))


def _int(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _check(got, q, k, v, bounds, what=""):
    """bounds: the (begin, end) of every sequence; the other rows of got must be zero."""
    Hq, g = q.shape[1], q.shape[1] // k.shape[1]
    rest = torch.ones(q.shape[0], dtype=torch.bool, device="cuda")
    for a, e in bounds:
        rest[a:e] = False
        seen = torch.ones((e - a, e - a), dtype=torch.bool, device="cuda").tril()
        for h in range(Hq):
            attn64.check(got[a:e, h], *attn64.attend(q[a:e, h], k[a:e, h // g], v[a:e, h // g], seen), (what, a, e, h))
    assert (got[rest] == 0).all(), what


def _bounds(lens, at=0):
    out = []
    for n in lens:
        out.append((at, at + n))
        at += n
    return out


@pytest.mark.parametrize("lens", [[1], [2], [31], [32], [33], [63], [64], [65], [127], [128], [129], [191], [256], [257], [1025],
                                  [1, 1, 1], [5, 0, 128, 0, 0, 129, 64], [0], [300, 1, 700]])
@pytest.mark.parametrize("D", [64, 128])
def test_lengths(lens, D):
    q, k, v = _inputs(sum(lens), 4, 2, D, sum(lens) + D)
    got = ops.prefill(q, k, v, _int([0] + [e for _, e in _bounds(lens)]))
    _check(got, q, k, v, _bounds(lens), lens)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (8, 8), (8, 1), (14, 2), (15, 3), (16, 4), (64, 8)])
def test_head_layouts(Hq, Hkv):
    lens = [200, 77]
    q, k, v = _inputs(277, Hq, Hkv, 128, Hq)
    _check(ops.prefill(q, k, v, _int([0, 200, 277])), q, k, v, _bounds(lens))


def test_many_short_sequences():
    """More sequences than a wave scans at once, and more than two rounds of it."""
    lens = [(7 * i) % 40 for i in range(150)]
    q, k, v = _inputs(sum(lens), 2, 1, 64, 3)
    b = _bounds(lens)
    _check(ops.prefill(q, k, v, _int([0] + [e for _, e in b])), q, k, v, b)


@pytest.mark.parametrize("D", [64, 128])
def test_slices_of_a_fused_projection(D):
    Hq, Hkv, lens = 6, 2, [130, 61]
    g = torch.Generator("cuda").manual_seed(9)
    x = torch.randn((191, Hq + 2 * Hkv, D), generator=g, device="cuda").half()
    q, k, v = x.split([Hq, Hkv, Hkv], 1)
    assert not q.is_contiguous()
    got = ops.prefill(q, k, v, _int([0, 130, 191]))
    assert torch.equal(got, ops.prefill(q.contiguous(), k.contiguous(), v.contiguous(), _int([0, 130, 191])))
    _check(got, q, k, v, _bounds(lens))


def test_head_major_and_shared_heads():
    """Heads outermost ([H, T, D] storage), and one K/V head expanded to several without a copy."""
    q, k, v = _inputs(150, 4, 2, 128, 11)
    cu = _int([0, 150])
    want = ops.prefill(q, k, v, cu)
    hm = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    assert torch.equal(ops.prefill(*hm, cu), want)
    k1, v1 = k[:, :1], v[:, :1]
    assert torch.equal(ops.prefill(q, k1.expand(-1, 4, -1), v1.expand(-1, 4, -1), cu), ops.prefill(q, k1.contiguous(), v1.contiguous(), cu))


def test_rows_of_no_sequence_are_zero():
    q, k, v = _inputs(400, 2, 2, 128, 5)
    got = ops.prefill(q, k, v, _int([70, 70, 201, 333]))
    _check(got, q, k, v, [(70, 201), (201, 333)])


def test_bounds_out_of_order_or_range():
    """A falling bound counts as its predecessor, one above the rows as their number, one below 0 as 0."""
    q, k, v = _inputs(300, 2, 1, 64, 6)
    got = ops.prefill(q, k, v, _int([-5, 100, 40, 250, 9999]))
    _check(got, q, k, v, [(0, 100), (100, 250), (250, 300)])


@pytest.mark.parametrize("scale", [0.0, 1e-3, 8.0, 60.0])
def test_flat_and_peaked_scores(scale):
    q, k, v = _inputs(333, 2, 1, 128, 7, scale)
    _check(ops.prefill(q, k, v, _int([0, 333])), q, k, v, [(0, 333)])


def test_rising_and_falling_scores():
    """A new maximum at nearly every position, and only ever smaller ones."""
    n, D = 520, 128
    q, k, v = _inputs(n, 1, 1, D, 8)
    q[:] = 1
    for sign in (1, -1):
        k[:] = (sign * torch.linspace(-6, 6, n, device="cuda"))[:, None, None].half()
        _check(ops.prefill(q, k, v, _int([0, n])), q, k, v, [(0, n)], sign)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_values_stay_in_their_sequence(bad):
    """NaN and infinities in one sequence, and in rows of none, leave the other sequences as they were."""
    q, k, v = _inputs(500, 2, 1, 128, 12)
    cu = _int([10, 200, 330, 480])
    want = ops.prefill(q, k, v, cu)
    for t in (q, k, v):
        t[200:330] = bad
        t[:10] = bad
        t[480:] = bad
    got = ops.prefill(q, k, v, cu)
    assert torch.equal(got[:200], want[:200]) and torch.equal(got[330:], want[330:])


@pytest.mark.parametrize("at", [1, 40, 127, 128, 200, 319])
def test_masked_keys_do_not_reach_earlier_rows(at):
    """NaN and infinities in row `at` of K leave the rows before it as they were."""
    q, k, v = _inputs(320, 2, 2, 128, 13)
    cu = _int([0, 320])
    want = ops.prefill(q, k, v, cu)
    for bad in (float("nan"), float("inf")):
        k[at] = bad
        assert torch.equal(ops.prefill(q, k, v, cu)[:at], want[:at]), bad


def test_infinite_scores():
    """A row whose scores are all -inf is zero; -inf scores among others drop out."""
    q, k, v = _inputs(100, 1, 1, 64, 14)
    q.abs_().clamp_(min=0.1)
    k[:] = -float("inf")
    assert (ops.prefill(q, k, v, _int([0, 100])) == 0).all()
    k[3] = 1.0
    got = ops.prefill(q, k, v, _int([0, 100]))
    assert (got[:3] == 0).all() and torch.equal(got[3:], v[3:4].expand(97, -1, -1))


def test_other_stream_and_graph():
    q, k, v = _inputs(300, 4, 2, 128, 15)
    cu = _int([0, 129, 300])
    want = ops.prefill(q, k, v, cu)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = ops.prefill(q, k, v, cu)
    st.synchronize()
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.prefill(q, k, v, cu)
    for i in range(3):
        q.normal_()
        cu.copy_(_int([0, 50 + i, 280]))
        eager = ops.prefill(q, k, v, cu)
        out.fill_(7)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), i


def test_c_abi_writes_its_rows_only():
    q, k, v = _inputs(140, 2, 1, 64, 16)
    cu = _int([0, 90, 140])
    buf = torch.full((160, 2, 64), 5.0, dtype=torch.float16, device="cuda")
    va.prefill(va.PrefillBufs(q.data_ptr(), k.data_ptr(), v.data_ptr(), cu.data_ptr(), buf[10:].data_ptr()),
               va.PrefillShape(2, 140, 2, 1, 64))
    torch.cuda.synchronize()
    assert (buf[:10] == 5).all() and (buf[150:] == 5).all()
    assert torch.equal(buf[10:150], ops.prefill(q, k, v, cu))


def test_empty_batch():
    q = torch.empty((0, 4, 128), dtype=torch.float16, device="cuda")
    assert ops.prefill(q, q[:, :2], q[:, :2], _int([0, 0])).shape == (0, 4, 128)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,at", [(1, 0), (50, 0), (50, 49), (130, 127), (130, 128), (300, 130), (700, 65), (700, 511)])
def test_infinite_and_nan_values_reach_the_rows_that_see_them_only(n, at, D):
    """Row `at` of V holds inf, -inf, NaN and finite values, as does row at + 3 (another order): a column's
    outputs are the values' sum from that row on, and as if both rows were finite before it."""
    q, k, v = _inputs(n, 2, 2, D, n + at)
    cu = _int([0, n])
    want = ops.prefill(q, k, v, cu)
    bad, kinds = v.clone(), torch.tensor([float("inf"), -float("inf"), float("nan"), 1.0], device="cuda").half()
    rows = [(at, 0)] + ([(at + 3, 1)] if at + 3 < n else [])
    for row, turn in rows:
        bad[row, 0] = kinds.roll(turn).repeat(D // 4)
    got = ops.prefill(q, k, bad, cu)
    assert torch.equal(got[:, 1], want[:, 1]) and torch.equal(got[:at], want[:at])
    odd = torch.zeros((n, D), dtype=torch.float64, device="cuda")
    for row, turn in rows:
        x = bad[row, 0].double()
        odd[row:] += torch.where(x.isfinite(), torch.zeros_like(x), x)
    x = got[:, 0].double()
    assert torch.equal(x.isnan(), odd.isnan())
    assert torch.equal(x == float("inf"), odd == float("inf")) and torch.equal(x == -float("inf"), odd == -float("inf"))


def test_infinite_and_nan_keys_reach_the_rows_that_see_them_only():
    for at in (0, 63, 140):
        q, k, v = _inputs(200, 2, 1, 128, at)
        cu = _int([0, 200])
        for x in (float("nan"), float("inf")):
            bad = k.clone()
            bad[at, 0, 5] = x
            got = ops.prefill(q, bad, v, cu)
            # not bit for bit: 32 rows take a new maximum together (an infinite score of one of them makes
            # them), which rounds a sum anew; what that may be off is part of the bound
            _check(got[:at], q[:at], k[:at], v[:at], [(0, at)])
            assert got[at:][(q[at:, :, 5] > 0)].isnan().all()        # a score of NaN, or of inf
