"""GPU: drafts behind the longest context that a block table can name, 2^31 - 64 positions with
them: positions, and the ends of the tiles around them, next to where 32 bits end. Every page but
the last is the same one."""
import pytest
import torch

import voltattn_amd.torch_ops  # noqa: F401

pytestmark = pytest.mark.gpu
ops = torch.ops.voltattn


@pytest.mark.parametrize("behind", [0, 60, 70])
def test_last_positions_of_32_bits(behind):
    """Drafts score 40 above a context of equal scores, which leaves it 2^31 / e^40 = 1e-8 of the weight:
    every draft's output is the mean of the values of the drafts that it sees."""
    T, D, page, pages = 8, 64, 64, (1 << 25) - 1
    n = pages * page - behind                               # the last tile of 128 is half full, or less, or full
    k = torch.zeros((3, 1, page, D), device="cuda")
    v = torch.full((3, 1, page, D), 3.0, device="cuda")
    place = [n - T + i for i in range(T)]
    last = {x: i for i, x in enumerate(sorted({p // page for p in place}), 1)}
    for i, p in enumerate(place):
        k[last[p // page], 0, p % page, 0] = 40.0
        v[last[p // page], 0, p % page] = float(i - 3)
    kp, ks = ops.quantize(k, 3, 64)
    vp, vs = ops.quantize(v, 3, 64)
    exact_k, exact_v = ops.dequantize(kp, ks, 3, 64), ops.dequantize(vp, vs, 3, 64)
    table = torch.zeros((1, pages), dtype=torch.int32, device="cuda")
    for p, i in last.items():
        table[0, p] = i
    q = torch.zeros((1, T, 1, D), dtype=torch.float16, device="cuda")
    q[..., 0] = 8.0                                         # 8 * 40 / sqrt(64)
    masks = [(1 << i) | (1 << (i // 2)) for i in range(T)]
    got = ops.decode_tree(q, kp, vp, ks, vs, table, torch.tensor([n - T], dtype=torch.int32, device="cuda"), None,
                          torch.tensor([masks], device="cuda"), "q3+", n, 64)[0, :, 0].double()
    at = [(last[p // page], p % page) for p in place]
    w = torch.tensor([float(exact_k[a, 0, r, 0]) for a, r in at], dtype=torch.float64, device="cuda").exp()
    x = torch.stack([exact_v[a, 0, r].double() for a, r in at])
    for i in range(T):
        seen = [j for j in range(T) if masks[i] >> j & 1]
        want = (w[seen, None] * x[seen]).sum(0) / w[seen].sum()
        # the weights' and the result's rounding, and the context's share
        assert ((got[i] - want).abs() <= 2.0 ** -11 * (x[seen].abs().amax() + want.abs()) + 1e-6).all(), i
