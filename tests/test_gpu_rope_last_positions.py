"""GPU: va_append_rope for rows around position 2^31: those behind the last one that a table could hold are not
written, and their q and k are turned by their own angle, as any others' are."""
import pytest
import torch

import voltattn_amd.torch_ops  # noqa: F401
from tests import block8
from tests.test_gpu_rope import Case, _copy, _int, _near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["b8+", "f16+", "q8+", "q3+"])
@pytest.mark.parametrize("new", [[3, 1, 9], [40, 70, 33]])      # few rows to a sequence, many
@pytest.mark.parametrize("interleaved", [False, True])
def test_positions_around_the_last_one(fmt, new, interleaved):
    c = Case(fmt, [0, 0, 0], new, G=32, seed=sum(new))
    start = [2 ** 31 - 2, 2 ** 31 - 1, 2 ** 31 - 40]
    before = _copy(c)
    q, k = c.run(start=_int(start), interleaved=interleaved)
    places = torch.tensor([s + i for s, n in zip(start, new) for i in range(n)], dtype=torch.int64, device="cuda")
    assert int(places.max()) >= 2 ** 31
    _near(q, *block8.rotate(c.q, places, c.freq, interleaved), "q")
    _near(k, *block8.rotate(c.k, places, c.freq, interleaved), "k")
    for old, now in zip(sum(before, []), c.pools + c.scales):
        assert old is None or torch.equal(old.view(torch.uint8), now.view(torch.uint8))
