"""GPU: pools whose later pages lie behind 2^32 bytes: the same results as from a small pool."""
import pytest
import torch

import voltattn_amd.torch_ops  # noqa: F401
from tests import block8

pytestmark = pytest.mark.gpu
ops = torch.ops.voltattn
HQ, HKV, D, PAGE, G = 8, 8, 128, 256, 32
FAR = (1 << 32) // (HKV * PAGE * D) + 20                          # pages: 5 GB of codes


def _int(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("new", [1, 40, 700])
def test_far_pages(new):
    g = torch.Generator("cuda").manual_seed(new)
    near = [torch.randn((6, HKV, PAGE, D), generator=g, device="cuda") for _ in "kv"]
    pools, scales = map(list, zip(*(block8.pack(x, G) for x in near)))
    far_p = [torch.empty((FAR, HKV, PAGE, D), dtype=torch.float8_e4m3fn, device="cuda") for _ in "kv"]
    far_s = [torch.zeros((FAR, HKV, PAGE // G), dtype=torch.float16, device="cuda") for _ in "kv"]
    for a, b in zip(far_p + far_s, pools + scales):
        a.view(torch.uint8)[-6:].copy_(b.view(torch.uint8))
    table = _int([[3, 0, 5, 1]])
    qkv = torch.randn((new, HQ + 2 * HKV, D), generator=g, device="cuda").half()
    freq = (10000.0 ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)).float()
    start, cu, lens = _int([300]), _int([0, new]), _int([300 + new])
    outs = []
    for t, p, s in ((table, pools, scales), (table + (FAR - 6), far_p, far_s)):
        q, _ = ops.append_rope(*qkv.split([HQ, HKV, HKV], 1), freq, cu, start, None, t, *p, *s, "b8+", G)
        outs.append((q, ops.attend_paged(q, *p, *s, t, cu, lens, "b8+", 4 * PAGE, G)))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    assert outs[0][1].isfinite().all() and (outs[0][1] != 0).any()
    for a, b in zip(far_p + far_s, pools + scales):
        assert torch.equal(a.view(torch.uint8)[-6:], b.view(torch.uint8))
