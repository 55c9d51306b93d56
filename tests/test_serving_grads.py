"""The serving operators have no gradients and say so: an output of prefill or decode_tree for
inputs that require grad raises in backward(), as that of decode_paged does, instead of leaving
gradients of None behind a warning. Inputs that require none, or calls under no_grad, are as they were."""
import warnings

import pytest
import torch

import voltattn_amd.torch_ops  # noqa: F401

ops = torch.ops.voltattn


def _int(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


def _calls(q_grad):
    g = torch.Generator("cuda").manual_seed(0)
    q = torch.randn((40, 4, 64), generator=g, device="cuda").half().requires_grad_(q_grad)
    k, v = (torch.randn((40, 2, 64), generator=g, device="cuda").half() for _ in "kv")
    yield q, lambda: ops.prefill(q, k, v, _int([0, 40]))
    qt = torch.randn((1, 3, 4, 64), generator=g, device="cuda").half().requires_grad_(q_grad)
    kp, vp = (torch.randn((2, 2, 64, 64), generator=g, device="cuda").half() for _ in "kv")
    yield qt, lambda: ops.decode_tree(qt, kp, vp, None, None, _int([[0, 1]]), _int([90]), None, _int([[1, 2, 4]], torch.int64), "f16+", 128)


@pytest.mark.gpu
def test_backward_raises():
    for leaf, call in _calls(True):
        out = call()
        assert out.requires_grad
        with pytest.raises(RuntimeError, match="no gradient|no autograd|autograd"):
            out.float().sum().backward()
        assert leaf.grad is None


@pytest.mark.gpu
def test_without_gradients_nothing_changes():
    plain = [call() for _, call in _calls(False)]
    assert not any(o.requires_grad for o in plain)
    with torch.no_grad():
        quiet = [call() for _, call in _calls(True)]
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        grads = [call() for _, call in _calls(True)]
    for a, b, c in zip(plain, quiet, grads):
        assert not b.requires_grad and torch.equal(a, b) and torch.equal(a, c.detach())


def test_traced_calls_raise_too():
    """The same through the shapes-only implementation (meta tensors)."""
    q = torch.empty((5, 4, 64), dtype=torch.float16, device="meta", requires_grad=True)
    k = torch.empty((5, 2, 64), dtype=torch.float16, device="meta")
    out = ops.prefill(q, k, k, torch.empty(2, dtype=torch.int32, device="meta"))
    assert out.shape == q.shape and out.requires_grad
    with pytest.raises(RuntimeError, match="no gradient|no autograd|autograd"):
        out.float().sum().backward()
    with torch.no_grad():
        assert not ops.prefill(q, k, k, torch.empty(2, dtype=torch.int32, device="meta")).requires_grad


@pytest.mark.gpu
def test_changed_pools_are_noticed():
    """A pool that backward() needs and that an operator then changes in place: torch's own error, no wrong gradient."""
    for change in ("compact", "fork", "resize"):
        pool = torch.ones((3, 1, 64, 64), device="cuda").half()
        x = torch.ones_like(pool).requires_grad_()
        table, refs = _int([[0, 1]]), _int([1, 1, 0])
        y = (x * pool).sum() + (torch.ones(3, device="cuda", requires_grad=True) * refs).sum()
        if change == "compact":
            ops.compact_kv(pool, pool.clone(), None, None, table, _int([0]), _int([[1]]), _int([1]), "f16+")
        elif change == "fork":
            ops.fork_pages(table, _int([100]), _int([0, 0]), refs, pool, pool.clone(), None, None, "f16+")
        else:
            ops.resize_pages(table, refs, _int([100]), _int([60]), 64)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()


@pytest.mark.gpu
def test_pools_made_in_inference_mode():
    """They keep no count of changes: the operators take them as they are."""
    with torch.inference_mode():
        pool = torch.ones((3, 1, 64, 64), device="cuda").half()
        table, refs = _int([[0, 1]]), _int([1, 1, 0])
    for again in (False, True):
        with torch.inference_mode(again):
            ops.compact_kv(pool, pool.clone(), None, None, table, _int([0]), _int([[1]]), _int([1]), "f16+")
            ops.fork_pages(table, _int([100]), _int([0]), refs, pool, pool.clone(), None, None, "f16+")
            assert int(ops.resize_pages(table, refs, _int([100]), _int([100]), 64)) == 0


@pytest.mark.gpu
def test_under_autocast_modes_and_compile():
    """The ways into the operators that do not take the plain call's short cut."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Through(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    for _, call in _calls(False):
        want = call()
        with torch.autocast("cuda"):
            assert torch.equal(call(), want)
        with Through():
            assert torch.equal(call(), want)
        with torch.inference_mode():
            assert torch.equal(call(), want)
    q = torch.randn((40, 4, 64), device="cuda").half()
    cu = _int([0, 40])
    traced = torch.compile(lambda x: ops.prefill(x, x[:, :2], x[:, 2:], cu) * 2, backend="aot_eager", fullgraph=True)
    assert torch.equal(traced(q), ops.prefill(q, q[:, :2], q[:, 2:], cu) * 2)
