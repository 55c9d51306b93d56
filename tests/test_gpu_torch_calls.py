"""GPU: the calls of append_rope and attend_paged that never reach Python (host/torch_calls.cpp) against
the ops that do the whole of a call in Python (append_rope_checked, attend_paged_checked): the same
results, counts of changes and errors."""
import pytest
import torch

import voltattn_amd.torch_ops  # noqa: F401
from tests.test_gpu_attend import Case as Attend
from tests.test_gpu_rope import BITS, Case as Rope

pytestmark = pytest.mark.gpu
ops = torch.ops.voltattn


def _rope_args(c, **kw):
    a = dict(q=c.q, k=c.k, v=c.v, freq=c.freq, cu=c.cu, start=torch.tensor(c.start, dtype=torch.int32, device="cuda"), positions=None,
             table=c.table, kp=c.pools[0], vp=c.pools[1], ks=c.scales[0], vs=c.scales[1], fmt=c.fmt, group=c.G, interleaved=False,
             rotated_k=True, scaling=1.0)
    a.update(kw)
    return a


def _fresh(a):
    a = dict(a)
    for n in ("kp", "vp", "ks", "vs"):
        a[n] = None if a[n] is None else a[n].clone()
    return a


def _same(op, checked, a):
    x, y = _fresh(a), _fresh(a)
    got, want = op(*x.values()), checked(*y.values())
    for g, w in zip(got, want):
        assert g.shape == w.shape and torch.equal(g, w)
    for n in ("kp", "vp", "ks", "vs"):
        if a[n] is not None:
            assert torch.equal(x[n].view(torch.uint8), y[n].view(torch.uint8)), n
            assert x[n]._version == y[n]._version == 1, n


@pytest.mark.parametrize("fmt", ["b8+", *BITS])
def test_append_rope(fmt):
    c = Rope(fmt, [0, 70, 5], [33, 1, 100], D=64, G=32, page=64, seed=1)
    a = _rope_args(c)
    places = torch.arange(134, dtype=torch.int32, device="cuda") * 7
    for kw in ({}, dict(interleaved=True, rotated_k=False), dict(positions=places, scaling=0.5), dict(freq=c.freq[:8].clone())):
        _same(ops.append_rope, ops.append_rope_checked, dict(a, **kw))
    one = Rope(fmt, [0, 70, 5], [1, 1, 1], D=128, G=64, page=128, seed=2)
    _same(ops.append_rope, ops.append_rope_checked, _rope_args(one, cu=None))


def test_append_rope_of_no_rows_and_in_inference_mode():
    c = Rope("b8+", [3], [1], seed=3)
    a = _rope_args(c)
    with torch.inference_mode():
        q, k = ops.append_rope(*dict(_fresh(a)).values())
    assert torch.equal(q, ops.append_rope_checked(*_fresh(a).values())[0])
    none = dict(q=c.q[:0], k=c.k[:0], v=c.v[:0], cu=torch.zeros(2, dtype=torch.int32, device="cuda"))
    x = _fresh(dict(a, **none))
    q, k = ops.append_rope(*x.values())
    assert q.shape == (0, 4, 128) and k.shape == (0, 2, 128) and torch.equal(x["kp"].view(torch.uint8), c.pools[0].view(torch.uint8))


@pytest.mark.parametrize("lens,new", [([300, 64, 1], [1, 1, 1]), ([700, 90], [520, 3])])
def test_attend_paged(lens, new):
    c = Attend(lens, new, seed=4)
    args = [c.q, *c.pools, *c.scales, c.table, c.cu, c.seq, "b8+", c.cap, c.G]
    assert torch.equal(ops.attend_paged(*args), ops.attend_paged_checked(*args))
    with torch.inference_mode():
        assert torch.equal(ops.attend_paged(*args), ops.attend_paged_checked(*args))


def _error(op, args):
    with pytest.raises((RuntimeError, ValueError)) as e:
        op(*args)
    return str(e.value).split("\n")[0]


def test_refusals_are_those_of_the_checked_ops():
    c = Attend([300, 64], [2, 1], seed=5)
    args = [c.q, *c.pools, *c.scales, c.table, c.cu, c.seq, "b8+", c.cap, c.G]
    for at, bad in [(0, c.q.float()), (0, c.q[:, :3]), (0, c.q.transpose(0, 1)), (1, c.pools[0].view(torch.uint8)), (2, c.pools[1][:, :1]),
                    (3, c.scales[0][..., :0]), (4, c.scales[1].cpu()), (5, c.table.long()), (5, c.table.t()), (6, c.cu[:2]), (6, None),
                    (7, c.seq[:1]), (8, "q8+"), (9, -1), (9, 1 << 40), (10, 48)]:
        x = list(args)
        x[at] = bad
        text = _error(ops.attend_paged, x)
        assert text == _error(ops.attend_paged_checked, x).replace("_checked", ""), (at, bad)
    r = Rope("b8+", [3, 0], [1, 2], seed=6)
    a = _rope_args(r)
    for name, bad in [("q", r.q.float()), ("q", r.q[..., ::2]), ("k", r.k[:2]), ("v", r.v.cpu()), ("freq", r.freq[:7]), ("freq", r.freq.half()),
                      ("cu", None), ("start", a["start"][:1]), ("positions", a["start"]), ("table", r.table.t()), ("kp", r.pools[0][:2]),
                      ("ks", None), ("vs", r.scales[1][..., :0]), ("fmt", "q5"), ("fmt", "q8+"), ("group", 16)]:
        x = _fresh(dict(a, **{name: bad}))
        text = _error(ops.append_rope, x.values())
        assert text == _error(ops.append_rope_checked, x.values()).replace("_checked", ""), (name, bad)
        assert torch.equal(x["vp"].view(torch.uint8), a["vp"].view(torch.uint8))


def test_gradients_are_refused():
    c = Attend([64], [1], seed=7)
    q = c.q.clone().requires_grad_()
    out = ops.attend_paged(q, *c.pools, *c.scales, c.table, c.cu, c.seq, "b8+", c.cap, c.G)
    assert out.requires_grad
    with pytest.raises(RuntimeError):
        out.sum().backward()
    with torch.no_grad():
        assert not ops.attend_paged(q, *c.pools, *c.scales, c.table, c.cu, c.seq, "b8+", c.cap, c.G).requires_grad
