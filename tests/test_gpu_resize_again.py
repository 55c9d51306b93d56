"""GPU: a growth that the pool could not serve is taken back by resizing to the old lengths: the table and
the counts are as before it, and a smaller one then succeeds."""
import pytest
import torch

import voltattn_amd.torch_ops  # noqa: F401
from tests.test_gpu_pages import Pool, _int, ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B", [3, 40])
def test_growth_taken_back(B):
    page, wide = 8, 6
    table = [[2 * b, 2 * b + 1] + [-1] * (wide - 2) for b in range(B)]
    refs = [1] * (2 * B) + [0] * (B + 1)
    m, t, r = Pool(table, refs, page), _int(table), _int(refs)
    old, new, less = [2 * page] * B, [4 * page] * B, [3 * page] * B
    missing = int(ops.resize_pages(t, r, _int(old), _int(new), page))
    assert missing == m.resize(old, new) == B - 1 and t.tolist() == m.table and r.tolist() == m.refs
    assert int(ops.resize_pages(t, r, _int(new), _int(old), page)) == 0
    assert t.tolist() == table and r.tolist() == refs
    assert int(ops.resize_pages(t, r, _int(old), _int(less), page)) == 0
    assert torch.equal(t[:, 2], torch.arange(2 * B, 3 * B, device="cuda", dtype=torch.int32))
