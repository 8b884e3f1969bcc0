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


def test_fork_into_what_it_reads(cuda):
    """Results that lie, in part, in the table, the lengths, the parents or each other are refused."""
    import torch
    from ivonar_amd import paging
    from ivonar_amd.runtime import KernelError

    pool = paging.page_pool(40, 64, cuda)
    ints = torch.full((60,), -1, dtype=torch.int32, device=cuda)
    table, lengths, parents, other = ints[:6].view(2, 3), ints[8:10].zero_(), ints[12:14].zero_(), ints[20:]
    apart = other[:6].view(2, 3), other[6:8]
    paging.fork(pool, table.clone(), lengths.clone(), parents, out=apart)
    for out in ((table, apart[1]), (apart[0], lengths), (apart[0], parents), (apart[0], ints[5:7]), (ints[9:15].view(2, 3), apart[1]),
                (ints[3:9].view(2, 3), apart[1]), (apart[0], other[5:7]), (apart[0], ints[13:15])):
        with pytest.raises(KernelError):
            paging.fork(pool, table, lengths, parents, out=out)
