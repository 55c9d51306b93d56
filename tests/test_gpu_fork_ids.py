"""GPU: va_fork_pages carries block-table entries outside the pool along, whatever their value, and
neither counts them nor gives them pages, by the plan of a small batch (one launch) and of a
large one (two), against the pool's model."""
import random

import pytest
import torch

import voltattn_amd.torch_ops  # noqa: F401
from tests.test_gpu_pages import Pool, _bytes, _int, _pools, _same, ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("odd", [-2, -1, -3, -(2 ** 31), 2 ** 31 - 1])
@pytest.mark.parametrize("B,wide", [(6, 5), (14, 5), (15, 5), (80, 5), (3, 9000)])
def test_ids_outside_the_pool_are_carried_along(B, wide, odd):
    rng = random.Random(B + wide)
    page, fmt, spare = 8, "q8+", 4 * B
    lens = [rng.randrange(0, min(wide, 5) * page + 1) for _ in range(B)]
    lens[0], lens[1] = 2 * page + 3, page                   # a page in part, and full ones only
    need = [-(-n // page) for n in lens]
    ids = list(range(sum(need) + spare))
    rng.shuffle(ids)
    table = [[ids.pop() for _ in range(n)] + [-1] * (wide - n) for n in need]
    refs = [1] * (sum(need) + spare)
    for i in ids:
        refs[i] = 0
    for b in range(B):                                      # every third last entry, some others
        if need[b] and b % 3 == 0:
            refs[table[b][need[b] - 1]] = 0
            table[b][need[b] - 1] = odd
        elif need[b] > 1 and b % 3 == 1:
            refs[table[b][0]] = 0
            table[b][0] = odd
    parents = [rng.randrange(B) for _ in range(B)] + [0, 0, 1]
    pools = _pools(fmt, len(refs), 2, page, 64, 32)
    want = [_bytes(t) for t in pools]
    m = Pool(table, refs, page)
    new_table, new_lens, missing, copies = m.fork(lens, parents)
    for src, to, n in copies:
        for w in want:
            w[to, :, :n] = w[src, :, :n]
    t, r = _int(table), _int(refs)
    got_table, got_lens, got_missing = ops.fork_pages(t, _int(lens), _int(parents), r, *pools, fmt, 32)
    assert got_table.tolist() == new_table and got_lens.tolist() == new_lens
    assert r.tolist() == m.refs and int(got_missing) == missing
    _same(pools, want)
