"""CPU: launches of 2^24 work-groups and more, whose 2^32 threads a launch does not count (a larger grid
runs as what is left of it modulo 2^32), are refused before any of them."""
import pytest

import voltattn_amd as va
from tests.test_serving_args import VA_ERANGE, _compact, _fork, _message, _prefill, _tree


@pytest.mark.parametrize("call,kw", [
    (_prefill, dict(B=1 << 18, total=1 << 18, Hq=64)),                       # 2^18 row tiles at least, 64 heads
    (_prefill, dict(B=1, total=(1 << 31) - 1, Hq=2)),
    (_compact, dict(B=(1 << 21) + 1)), (_compact, dict(B=1 << 21)),          # 8 K/V heads each
    (_fork, dict(children=(1 << 21) + 1)), (_fork, dict(children=1 << 21)),
    (_tree, dict(fmt="f16+", T=1, B=1 << 21, Hq=8, max_seq_len=1)),
])
def test_grids(call, kw):
    assert call(**kw) == VA_ERANGE
    assert "too" in _message()


def test_tree_workspace_of_refused_batches():
    from tests.test_serving_args import _shape
    s = _shape(B=1 << 21, Hq=8, max_seq_len=1)
    assert va.lib.va_tree_ws_bytes(int(va.Fmt.F16M), s, 1) == 0
