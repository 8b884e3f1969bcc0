"""Counts of slots that lie far past a table."""

from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sequences,width,page,free", [(1, 3, 32, 64), (3, 1, 64, 2), (70, 5, 32, 1000), (1500, 2, 32, 100)])
def test_slots_far_past_the_table(cuda, sequences, width, page, free):
    """Each sequence lacks up to 2^26 slots; their number is right up to the largest that the result holds."""
    import torch
    from ivonar_amd import paging

    for length, count in ((0, 2 ** 31 - 1), (page * width, 2 ** 31 - 1), (2 ** 30, 2 ** 30), (7, page * (1 << 20)),
                          (2 ** 31 - 1, 2 ** 31 - 1)):
        pool = paging.page_pool(free, page, cuda)
        table = torch.full((sequences, width), -1, dtype=torch.int32, device=cuda)
        ints = [torch.full((sequences,), value, dtype=torch.int32, device=cuda) for value in (length, count)]
        slots = -(-(length + count) // page) - -(-length // page)
        inside = max(0, width - -(-length // page))
        given = min(free, sequences * inside)
        missing = paging.reserve(pool, table, *ints)
        assert int(missing) == min(sequences * slots - given, 2 ** 31 - 1)
        assert int((table >= 0).sum()) == int(pool.refs.sum()) == given
