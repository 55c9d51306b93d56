"""GPU: va_attend_paged over batches so large that beginning a block counts in the shares, and that shares go by the
work-groups' ages, in the forms of 16, 32, 128 and 256 rows to a block, against float64 (attn_bound's bound); with
sequences of no rows, of one and with lengths out of range among them."""
import pytest
import torch

import voltattn_amd.torch_ops  # noqa: F401
from tests.test_gpu_attend import Case

pytestmark = pytest.mark.gpu


def _plan(c):
    """(rows to a block, tiles that the host counts to a work-group, real tiles to a work-group)."""
    B, total, group = len(c.lens), sum(c.new), c.Hq // c.Hkv
    mean = total * group / B
    rows = 16 if mean <= 16 else 32 if mean <= 32 else 128 if mean <= 2048 else 256
    bn = 64 if rows >= 128 else 128
    most = min(total * group, total * group // rows + B + 2) * c.Hkv * -(-c.cap // bn)
    groups = min(most, (3 if rows == 128 else 2) * torch.cuda.get_device_properties(0).multi_processor_count)
    real = 0
    for n, t in zip(c.lens, c.new):
        for rb in range(-(-t * group // rows)):
            last = min(t - 1, (rb * rows + rows - 1) // group)
            real += max(1, -(-(n - t + last + 1) // bn)) * c.Hkv
    return rows, most // groups, real / groups


def _run(c, rows, ages, bad=()):
    assert _plan(c)[0] == rows and _plan(c)[1] >= 8              # what beginning a block costs is counted
    assert not ages or _plan(c)[2] >= 17                         # shares go by age
    seq = c.seq.clone()
    for b in bad:
        seq[b] = c.cap + 1
    got = c.run(seq=seq)
    c.check(got, skip=bad)
    for b in bad:
        assert got[sum(c.new[:b]):sum(c.new[:b + 1])].isnan().all()
    assert torch.equal(c.run(seq=seq).view(torch.int16), got.view(torch.int16))


@pytest.mark.parametrize("D,G", [(64, 32), (128, 64)])
@pytest.mark.parametrize("new,group,rows", [(1, 2, 16), (3, 8, 32)])
def test_few_rows(D, G, new, group, rows):
    lens = [(i * 389) % 2500 + new for i in range(64)]
    c = Case(lens, [new if i % 9 else 0 for i in range(64)], 4 * group, 4, D, G, 64, seed=D)
    _run(c, rows, False, bad=(4, 40))


@pytest.mark.parametrize("D,G", [(64, 64), (128, 32)])
@pytest.mark.parametrize("lens,new,bad", [
    ([3000, 6000, 1200], [500, 700, 300], ()),
    ([4000, 64, 2900, 5000, 700, 40, 3300], [600, 1, 800, 400, 0, 40, 500], (1,)),
])
def test_many_rows(D, G, lens, new, bad):
    _run(Case(lens, new, 32, 8, D, G, 128, seed=sum(new)), 128, True, bad)


@pytest.mark.parametrize("D,G", [(64, 32), (64, 64), (128, 32), (128, 64)])
@pytest.mark.parametrize("lens,new,bad", [([6000, 3500], [900, 700], ()), ([4100, 2500, 3000], [1500, 130, 1400], (1,))])
def test_very_many_rows(D, G, lens, new, bad):
    _run(Case(lens, new, 32, 8, D, G, 256, seed=sum(new)), 256, True, bad)


@pytest.mark.parametrize("lens,new", [([700, 800], [700, 520]), ([513], [512]), ([3000, 900], [257, 900]), ([1100, 70], [1090, 1])])
def test_long_chunks(lens, new):
    """Blocks of 256 rows of 64 dimensions with a scale for 32 positions, whole and in part."""
    c = Case(lens, new, 16, 2, 64, 32, 128, seed=sum(new))
    c.check(c.run())
