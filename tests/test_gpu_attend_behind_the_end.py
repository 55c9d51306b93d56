"""GPU: va_attend_paged gives the same bits whatever finite scales lie behind a sequence's last position, in its
last tile's other half among them: a page's earlier owner may have left any."""
import pytest
import torch

import voltattn_amd.torch_ops  # noqa: F401
from tests.test_gpu_attend import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("G", [32, 64])
@pytest.mark.parametrize("lens,new", [([20, 31, 32, 84], [1, 1, 1, 1]), ([30, 70], [6, 6]), ([20, 32, 90, 1, 160], [20, 31, 60, 1, 160]),
                                      ([600, 532], [600, 532])])
@pytest.mark.parametrize("own", [2.0 ** -24, 2.0 ** -9, 2.0 ** 15])
def test_scales_behind_the_last_position(lens, new, G, own):
    c = Case(lens, new, 8, 2, 128, G, 64, seed=sum(lens))
    c.scales[1].fill_(own)
    if own > 1:
        c.pools[1].view(torch.uint8).bitwise_and_(0x87)          # codes below 2^-6: the output fits fp16
    want = c.run()
    c.check(want)
    for behind in (2.0 ** 15, 2.0 ** -24, 0.0, 37.51, -65504.0, 5 * 2.0 ** -24):
        for b, n in enumerate(lens):
            page, row = c.host[b][(n - 1) // 64], (n - 1) % 64 + 1
            for s in c.scales:
                s[page, :, -(-row // G):] = behind
        assert torch.equal(c.run(), want), behind
