"""GPU: NaN codes of V in batches where every work-group of the few rows' form has several pieces, one
behind the other: a piece's codes that were left out reach the rows that see them, whichever of its
waves has them and whatever the piece before it left out, and no others."""
import pytest
import torch

import voltattn_amd.torch_ops  # noqa: F401
from tests.test_gpu_attend import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,group", [(1, 4), (3, 8)])           # 16 rows to a block, 32
@pytest.mark.parametrize("D", [64, 128])
def test_every_wave_of_every_piece(n, group, D):
    B, Hkv = 700, 2
    lens = [97 + (i * 11) % 32 if i % 5 else 33 + (i * 7) % 96 for i in range(B)]
    c = Case(lens, [n] * B, group * Hkv, Hkv, D, 32, 64, seed=D + n)
    want = c.run()
    assert want.isfinite().all()
    v = c.pools[1].view(torch.uint8)
    expect = want.clone()
    for b in range(B):
        if b % 3 == 2:
            continue
        # in the last 32 positions' part (the wave that does not see all of it), or two parts with one
        for p, head, dim in [(lens[b] - 1 - b % 2, b % Hkv, b % D)] + ([(lens[b] - n, 1 - b % Hkv, (b + 9) % D)] if b % 4 == 0 else []):
            v[c.host[b][p // 64], head, p % 64, dim] = 0x7F if b % 2 else 0xFF
            first = b * n + max(0, p - (lens[b] - n))               # the rows from the position's own on
            expect[first:(b + 1) * n, head * group:(head + 1) * group, dim] = float("nan")
    assert expect.isnan().any() and not expect.isnan().all()
    for _ in range(5):
        got = c.run()
        assert torch.equal(got.isnan(), expect.isnan())
        assert torch.equal(got.nan_to_num(), expect.nan_to_num())
