"""GPU: va_attend_paged over batches of more than 64 sequences with many rows each, with sequences
without rows and lengths out of range among them, against float64 (attn_bound's bound)."""
import random

import pytest
import torch

import voltattn_amd.torch_ops  # noqa: F401
from tests.test_gpu_attend import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,n,longest", [(65, 14, 300), (130, 12, 200), (200, 9, 150), (70, 40, 900)])
def test_many_rows_of_many_sequences(B, n, longest):
    r = random.Random(B + n)
    new = [r.choice([0, 1, n, 2 * n]) for _ in range(B)]
    new[r.randrange(B)] = longest
    lens = [t + r.randint(0, 400) for t in new]
    bad = [i for i in r.sample(range(B), 5) if new[i]]
    c = Case(lens, new, 8, 1, 64, 32, 64, seed=B)
    seq = c.seq.clone()
    for j, b in enumerate(bad):
        seq[b] = [-1, c.cap + 1, -2 ** 31, 2 ** 31 - 1, c.cap + 64][j]
    got = c.run(seq=seq)
    c.check(got, skip=bad)
    for b in bad:
        at = sum(new[:b])
        assert got[at:at + new[b]].isnan().all()
    again = c.run(seq=seq)
    assert torch.equal(got.view(torch.int16), again.view(torch.int16))


@pytest.mark.parametrize("rows", [[40] * 3, [200] * 2 + [0] * 70, [0] * 66 + [300], [1] * 63 + [500, 0, 7]])
def test_rows_behind_and_before(rows):
    """Bounds that leave rows before the first and behind the last sequence."""
    c = Case([n + 77 for n in rows], rows, 8, 2, 128, 64, 64, seed=len(rows))
    want = c.run()
    q = torch.cat([c.q.new_full((5, 8, 128), 9), c.q, c.q.new_full((130, 8, 128), 9)])
    got = c.run(q=q, cu=c.cu + 5)
    assert (got[:5] == 0).all() and (got[5 + sum(rows):] == 0).all()
    c.check(got[5:5 + sum(rows)])
    c.check(want)
