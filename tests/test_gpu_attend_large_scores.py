"""GPU: va_attend_paged where scores are so large that a step of fp32 is a power of two or more: finite
queries, codes and scales give finite rows, which are the mean of the values whose scores are the
largest. Forms of 16, 32, 128 and 256 rows to a block.

What a row may be off is derived without its scores' own errors: in the first test a row's scores
are equal (the same operands in the same order, so equal in any arithmetic), in the second the largest
one is ahead of the others by more than both may be off and 40 powers of two."""
import math

import pytest
import torch

import voltattn_amd.torch_ops  # noqa: F401
from tests import attn_bound, block8
from tests.test_gpu_attend import Case

pytestmark = pytest.mark.gpu
ROWS = [(1, 900), (6, 700), (140, 800), (600, 1000)]           # new rows (4 query heads each), positions


def _rows(c, h, n):
    return [block8.rows(block8.values(p, s), c.host[0], n, h) for p, s in zip(c.pools, c.scales)]


@pytest.mark.parametrize("D,G", [(64, 32), (128, 64)])
@pytest.mark.parametrize("new,n", ROWS)
@pytest.mark.parametrize("size,scale", [(16.0, 2.0 ** 10), (512.0, 2.0 ** 14), (512.0, 25000.0), (8192.0, 2.0 ** 15), (16000.0, 40000.0)])
def test_equal_scores(new, n, D, G, size, scale):
    """All keys are the same row: the mean of what a row sees, for scores of 2^10 to 2^31 and below -2^31."""
    c = Case([n], [new], 8, 2, D, G, 64, seed=new + D)
    g = torch.Generator("cuda").manual_seed(new)
    key = torch.tensor([0x38, 0xB8, 0x3A, 0xB4], device="cuda", dtype=torch.uint8)[torch.randint(0, 4, (D,), generator=g, device="cuda")]
    c.pools[0].view(torch.uint8).copy_(key.expand(c.pools[0].shape))
    c.scales[0].fill_(scale)
    # values whose scales are powers of two, then any
    for any_scale in (False, True):
        if any_scale:
            c.scales[1].copy_(torch.rand(c.scales[1].shape, generator=g, device="cuda") * 0.01 + 0.001)
        c.q = (torch.randn(c.q.shape, generator=g, device="cuda") * size).clamp(-65504, 65504).half()
        got = c.run()
        assert got.isfinite().all()
        seen = torch.arange(n, device="cuda") <= (n - new + torch.arange(new, device="cuda"))[:, None]
        for h in range(2):
            k, v = _rows(c, h, n)
            out, bound = attn_bound.attend(torch.zeros((new, D), device="cuda"), k, v, seen)
            for i in range(4 * h, 4 * h + 4):
                off = (got[:, i].double() - out).abs()
                assert (off <= bound).all(), (i, any_scale, float((off / bound).max()))


@pytest.mark.parametrize("D,G", [(64, 64), (128, 32)])
@pytest.mark.parametrize("new,n", ROWS)
@pytest.mark.parametrize("size,scale", [(64.0, 2.0 ** 9), (256.0, 2.0 ** 14), (1024.0, 23456.0), (16000.0, 2.0 ** 15)])
def test_one_score_far_ahead(new, n, D, G, size, scale):
    """The value of the largest score: off by the weight's rounding (2^-11), that of the sum and quotient in fp32
    (2^-20 for all positions) and the result's (2^-11, or 2^-25)."""
    c = Case([n], [new], 8, 2, D, G, 64, seed=new + D + 1)
    g = torch.Generator("cuda").manual_seed(new + 1)
    c.scales[0].copy_(scale * torch.exp2(torch.randint(-2, 1, c.scales[0].shape, generator=g, device="cuda").float()))
    c.q = (torch.randn(c.q.shape, generator=g, device="cuda") * size).clamp(-65504, 65504).half()
    got = c.run()
    assert got.isfinite().all()
    seen = torch.arange(n, device="cuda") <= (n - new + torch.arange(new, device="cuda"))[:, None]
    sure = 0
    for h in range(2):
        k, v = _rows(c, h, n)
        for i in range(4 * h, 4 * h + 4):
            f = math.log2(math.e) / math.sqrt(D)
            s = (c.q[:, i].double() @ k.T * f).masked_fill(~seen, -math.inf)
            raw = (c.q[:, i].double().abs() @ k.abs().T * f).masked_fill(~seen, 0).amax(-1)
            top = s.topk(2, -1)
            ok = top.values[:, 0] - top.values[:, 1] > 2 * (D + 4) * 2.0 ** -24 * raw + 40
            sure += int(ok.sum())
            want = v[top.indices[:, 0]]
            off = (got[:, i].double() - want).abs()
            assert (off <= (2 * 2.0 ** -11 + 2.0 ** -20) * want.abs() + 2.0 ** -25 + 2.0 ** -30 * v.abs().max())[ok].all(), i
    assert sure >= 0.9 * new * 8, sure
