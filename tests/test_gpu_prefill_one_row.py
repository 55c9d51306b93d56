"""GPU: prompts of one row, whose row stride is never stepped: any slice of one row is taken,
also one from storage with heads outermost and far apart, and out of a longer tensor."""
import pytest
import torch

import voltattn_amd.torch_ops  # noqa: F401

pytestmark = pytest.mark.gpu
ops = torch.ops.voltattn


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows", [1, 2])
def test_slices_of_head_major_storage(rows, D):
    far = (1 << 24) // D // 8 + 8                           # 8 heads of it: more than 2^24 elements
    x = torch.randn((8, far, D), device="cuda").half().transpose(0, 1)[5:5 + rows]
    q = torch.randn((rows, 16, D), device="cuda").half()
    cu = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    want = ops.prefill(q, x.contiguous(), x.contiguous(), cu)
    assert torch.equal(ops.prefill(q, x, x, cu), want)
    wide = torch.randn((8 * 2, far, D), device="cuda").half().transpose(0, 1)[:rows]
    assert torch.equal(ops.prefill(wide, x, x, cu), ops.prefill(wide.contiguous(), x, x, cu))
    if rows == 1:                                           # softmax over one row: its values
        assert torch.equal(want, x.repeat_interleave(2, 1))


def test_one_row_expanded_in_heads():
    q, k = torch.randn((1, 4, 128), device="cuda").half(), torch.randn((1, 1, 128), device="cuda").half()
    cu = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    assert torch.equal(ops.prefill(q, k.expand(1, 4, 128), k.expand(1, 4, 128), cu), k.expand(1, 4, 128))
