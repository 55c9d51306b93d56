"""GPU: attention whose output comes from weights far below the largest one and from small
values (a sink: one position that takes most of the weight and has next to no value), by
the prompt kernel and by the tree kernel in every tiled format and row block. The bound is the
operator's (attn_bound.py), and none that an output of zeros would meet."""
import pytest
import torch

import voltattn_amd as va
import voltattn_amd.torch_ops  # noqa: F401
from tests import attn_bound

pytestmark = pytest.mark.gpu
ops = torch.ops.voltattn
BITS = {"f16+": 16, "q8+": 8, "q4+": 4, "q3+": 3}
FORMS = {32: (8, 4, 1), 64: (33, 4, 1), 128: (33, 4, 2)}     # query rows to a work-group: T, group, K/V heads


def _int(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


def _draws(n, heads, D, nats, spread, vmag, seed, rows, sink=0.01):
    """fp16 q [rows, heads.., D] and k, v [n, heads, D]: position 0 scores `nats` above the others, whose
    scores are N(0, spread^2), and has `sink` of their values, vmag * (1 + N(0, 1))."""
    g = torch.Generator("cuda").manual_seed(seed)
    q = torch.randn(rows + (D,), generator=g, device="cuda")
    k = torch.randn((n, heads, D), generator=g, device="cuda") * spread
    v = (torch.randn((n, heads, D), generator=g, device="cuda") + 1) * vmag
    q[..., 0] = 8
    k[..., 0] = 0
    k[0] = 0
    k[0, :, 0] = nats * D ** 0.5 / 8
    v[0] *= sink
    return q.half(), k.half(), v.half()


def _pools(fmt, rows, page, G):
    """[n, heads, D] as a pool of pages in order, its scales, and the values that these stand for [n, heads, D]."""
    n, heads, D = rows.shape
    pages = -(-n // page)
    x = torch.zeros((pages * page, heads, D), dtype=torch.float16, device="cuda")
    x[:n] = rows
    x = x.view(pages, page, heads, D).transpose(1, 2).contiguous()
    if fmt == "f16+":
        return x, None, rows
    pay, sc = ops.quantize(x.float(), BITS[fmt], G)
    return pay, sc, ops.dequantize(pay, sc, BITS[fmt], G).transpose(1, 2).reshape(-1, heads, D)[:n]


def _assert_form(fmt, form, n, D, G, page):
    """The workspace is two pieces of a row block for each work-group: those of this form."""
    T, group, heads = FORMS[form]
    shape = va.PagedShape(1, heads * group, heads, D, G, page, -(-(n + T) // page), -(-(n + T) // page), n + T)
    f = {"f16+": va.Fmt.F16M, "q8+": va.Fmt.Q8M, "q4+": va.Fmt.Q4M, "q3+": va.Fmt.Q3M}[fmt]
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    tiles = heads * -(-T * group // form) * -(-(n + T) // (128 if form == 32 else 64))
    groups = {32: min(2 * cus, tiles), 64: min(cus, tiles), 128: (3 if D == 128 or fmt == "f16+" else 4) * cus}[form]
    assert va.tree_ws_bytes(f, shape, T) == 2 * groups * form * (D + 2) * 4, "another row block"


def _tree(fmt, form, n, nats, spread, vmag, D=128, G=32, seed=0, sink=0.01):
    T, group, heads = FORMS[form]
    q, k, v = _draws(n + T, heads, D, nats, spread, vmag, seed, (1, T, heads * group), sink)
    page = 256
    _assert_form(fmt, form, n, D, G, page)
    kp, ks, kx = _pools(fmt, k, page, G)
    vp, vs, vx = _pools(fmt, v, page, G)
    table = _int([list(range(kp.shape[0]))])
    mask = _int([[1 << i if i < 63 else -(1 << 63) for i in range(T)]], torch.int64)
    got = ops.decode_tree(q, kp, vp, ks, vs, table, _int([n]), None, mask, fmt, n + T, G)[0]
    seen = torch.cat([torch.ones((T, n), dtype=torch.bool, device="cuda"), torch.eye(T, dtype=torch.bool, device="cuda")], 1)
    rounded = fmt != "f16+" and form == 128
    for h in range(heads * group):
        attn_bound.check(got[:, h], *attn_bound.attend(q[0, :, h], kx[:, h // group], vx[:, h // group], seen, rounded), h)


@pytest.mark.parametrize("vmag", [1.0, 0.02, 0.005, 0.0005])
@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("fmt", list(BITS))
def test_tree_with_a_sink(fmt, form, vmag):
    _tree(fmt, form, 16384, 12.0, 1.0, vmag)


@pytest.mark.parametrize("nats", [6.0, 16.0])
@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("fmt", list(BITS))
def test_tree_with_a_sink_over_equal_scores(fmt, form, nats):
    """Equal weights round alike: nothing averages out."""
    _tree(fmt, form, 16384, nats, 0.0, 1.0, seed=1, sink=0.0)


@pytest.mark.parametrize("D,G", [(128, 64), (64, 32), (64, 64)])
@pytest.mark.parametrize("fmt", ["q8+", "q4+", "q3+"])
def test_tree_with_a_sink_in_the_other_row_layouts(fmt, D, G):
    for form in (32, 64):
        _tree(fmt, form, 8192, 10.0, 1.0, 0.01, D, G, seed=2)


@pytest.mark.parametrize("form", [32, 64])
@pytest.mark.parametrize("fmt", ["q8+", "q4+", "q3+"])
def test_tree_over_values_of_very_different_size(fmt, form):
    """Values that grow with the position, by 2^16 over the context, and that fall: the sums follow the
    largest scale so far."""
    T, group, heads = FORMS[form]
    n, D, G, page = 3000, 128, 32, 256
    for sign in (1, -1):
        q, k, v = _draws(n + T, heads, D, 2.0, 1.0, 1.0, 3, (1, T, heads * group))
        v = (v.float() * torch.exp2(sign * torch.linspace(-8, 8, n + T, device="cuda"))[:, None, None]).half()
        kp, ks, kx = _pools(fmt, k, page, G)
        vp, vs, vx = _pools(fmt, v, page, G)
        mask = _int([[1 << i for i in range(T)]], torch.int64)
        got = ops.decode_tree(q, kp, vp, ks, vs, _int([list(range(kp.shape[0]))]), _int([n]), None, mask, fmt, n + T, G)[0]
        seen = torch.cat([torch.ones((T, n), dtype=torch.bool, device="cuda"), torch.eye(T, dtype=torch.bool, device="cuda")], 1)
        for h in range(heads * group):
            attn_bound.check(got[:, h], *attn_bound.attend(q[0, :, h], kx[:, h // group], vx[:, h // group], seen), (sign, h))


@pytest.mark.parametrize("nats,spread", [(6.0, 0.0), (16.0, 0.0), (12.0, 1.0)])
@pytest.mark.parametrize("D", [64, 128])
def test_prompt_with_a_sink(D, nats, spread):
    n, heads = 4097, 2
    q, k, v = _draws(n, heads, D, nats, spread, 1.0, 4, (n, heads), 0.0)
    got = ops.prefill(q, k, v, _int([0, n]))
    rows = torch.arange(1024, n, 96, device="cuda")         # rows with a tail in their outputs
    seen = torch.arange(n, device="cuda")[None] <= rows[:, None]
    for h in range(heads):
        attn_bound.check(got[rows, h], *attn_bound.attend(q[rows, h], k[:, h], v[:, h], seen), h)
