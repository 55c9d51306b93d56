"""The operators have no forward-mode gradients either and say so: a tensor with a tangent raises, instead of
giving an output without one (test_serving_grads.py has backward())."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import voltattn_amd.torch_ops  # noqa: F401

ops = torch.ops.voltattn


def _calls(device):
    """name, the tensors that may have tangents, and the call with them."""
    half = lambda *s: torch.zeros(s, dtype=torch.float16, device=device)                 # noqa: E731
    ints = lambda *s: torch.zeros(s, dtype=torch.int32, device=device)                   # noqa: E731
    code = lambda: torch.zeros((2, 2, 64, 64), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)   # noqa: E731
    cu, table = ints(2), ints(1, 2)
    yield "prefill", [half(5, 4, 64), half(5, 2, 64), half(5, 2, 64)], lambda q, k, v: ops.prefill(q, k, v, cu)
    yield ("decode_tree", [half(1, 3, 4, 64), half(2, 2, 64, 64), half(2, 2, 64, 64)],
           lambda q, k, v: ops.decode_tree(q, k, v, None, None, table, ints(1), None, torch.zeros((1, 3), dtype=torch.int64, device=device), "f16+", 128))
    yield ("append_rope", [half(5, 4, 64), half(5, 2, 64), half(5, 2, 64), torch.zeros(32, device=device)],
           lambda q, k, v, f: ops.append_rope(q, k, v, f, cu, ints(1), None, table, code(), code(), half(2, 2, 2), half(2, 2, 2), "b8+", 32, False, True)[0])
    yield ("append_rope", [half(5, 4, 64), half(2, 2, 64, 64), half(2, 2, 64, 64)],
           lambda q, k, v: ops.append_rope(q, half(5, 2, 64), half(5, 2, 64), torch.zeros(32, device=device), cu, ints(1), None, table, k, v, None, None, "f16+")[0])
    yield ("attend_paged", [half(5, 4, 64), half(2, 2, 2), half(2, 2, 2)],
           lambda q, sk, sv: ops.attend_paged(q, code(), code(), sk, sv, table, cu, ints(1), "b8+", 128, 32))


def _check(device):
    for name, args, call in _calls(device):
        plain = call(*args)
        with fwd.dual_level():
            assert fwd.unpack_dual(call(*args)).tangent is None                          # none to lose
            for i in range(len(args)):
                x = list(args)
                x[i] = fwd.make_dual(args[i].clone(), torch.ones_like(args[i]))
                for quiet in (False, True):
                    with torch.set_grad_enabled(not quiet), pytest.raises(RuntimeError, match=f"{name}.*no gradient"):
                        call(*x)
        with pytest.raises(RuntimeError, match=f"{name}.*no gradient"):
            torch.func.jvp(call, tuple(args), tuple(torch.ones_like(a) for a in args))
        assert call(*args).shape == plain.shape


def test_tangents_are_refused_where_only_shapes_are_made():
    _check("meta")


@pytest.mark.gpu
def test_tangents_are_refused():
    _check("cuda")
