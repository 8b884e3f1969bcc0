"""The page pool against a plain implementation, number for number, and the copies' bytes."""

from __future__ import annotations

import numpy as np
import pytest

import _paging

pytestmark = pytest.mark.gpu


def _ints(cuda, values):
    import torch

    return torch.from_numpy(np.ascontiguousarray(values, dtype=np.int32)).to(cuda)


class Both:
    """The device's pool and table and the plain ones, the same calls on either."""

    def __init__(self, cuda, pages, page_size, sequences, width):
        import torch
        from ivonar_amd import paging

        self.paging, self.cuda = paging, cuda
        self.pool, self.plain = paging.page_pool(pages, page_size, cuda), _paging.Pool(pages, page_size)
        self.table = torch.full((sequences, width), -1, dtype=torch.int32, device=cuda)
        self.expected = np.full((sequences, width), -1, dtype=np.int32)

    def check(self, what=""):
        assert np.array_equal(self.table.cpu().numpy(), self.expected), what
        assert np.array_equal(self.pool.refs.cpu().numpy(), self.plain.refs), what
        assert np.array_equal(self.pool.free.cpu().numpy(), self.plain.words()), what

    def reserve(self, lengths, counts):
        missing = self.paging.reserve(self.pool, self.table, _ints(self.cuda, lengths), _ints(self.cuda, counts))
        assert int(missing) == self.plain.reserve(self.expected, lengths, counts)
        self.check("reserve")
        return int(missing)

    def release(self, first=None, last=None):
        self.paging.release(self.pool, self.table, *(None if x is None else _ints(self.cuda, x) for x in (first, last)))
        self.plain.release(self.expected, first, last)
        self.check("release")

    def fork(self, lengths, parents):
        fork = self.paging.fork(self.pool, self.table, _ints(self.cuda, lengths), _ints(self.cuda, parents))
        self.expected, new_lengths, copies, missing = self.plain.fork(self.expected, lengths, parents)
        self.table = fork.table
        self.check("fork")
        assert np.array_equal(fork.lengths.cpu().numpy(), new_lengths) and int(fork.missing) == missing
        listed = fork.copies.cpu().numpy()
        assert [tuple(c) for c in listed[:len(copies)].tolist()] == copies and (listed[len(copies):] == -1).all()
        return new_lengths, fork.copies

    def compact(self):
        copies, held = self.paging.compact(self.pool, self.table)
        expected, count = self.plain.compact(self.expected)
        self.check("compact")
        assert int(held) == count
        listed = copies.cpu().numpy()
        assert [tuple(c) for c in listed[:len(expected)].tolist()] == expected and (listed[len(expected):] == -1).all()
        return copies


@pytest.mark.parametrize("pages", [1, 31, 32, 33, 100, 1000])
def test_new_pool(cuda, pages):
    both = Both(cuda, pages, 64, 2, 3)
    both.check()
    both.compact()
    both.release()


@pytest.mark.parametrize("pages,sequences,width,page", [(200, 5, 30, 32), (33, 1, 40, 64), (3000, 130, 20, 128),
                                                        (2500, 1100, 3, 32), (40000, 4, 9000, 32)])
def test_calls_one_after_another(cuda, pages, sequences, width, page):
    """Sequences that grow, shrink, lose their first pages, fork, end and move together, many times."""
    rng = np.random.default_rng(pages)
    both = Both(cuda, pages, page, sequences, width)
    lengths = np.zeros(sequences, dtype=np.int64)
    for turn in range(12):
        room = width * page - lengths
        counts = np.minimum(rng.integers(0, max(2, 2 * pages * page // max(1, sequences * 6)), len(lengths)), room)
        counts[rng.random(len(lengths)) < 0.3] = 1
        counts = np.minimum(counts, room)
        if both.reserve(lengths, counts):
            both.release(last=np.where(rng.random(len(lengths)) < 0.5, width, 0))
            lengths = np.where((both.expected >= 0).any(1), lengths, 0)
            lengths = np.minimum(lengths, ((both.expected >= 0).sum(1)) * page)
        else:
            lengths = lengths + counts
        if turn % 3 == 1:  # tokens dropped from the end, and pages before a window
            lengths = np.maximum(0, lengths - rng.integers(0, 3 * page, len(lengths)))
            both.release(first=-(-lengths // page))
            both.release(last=np.maximum(0, lengths - 5 * page) // page)
        if turn % 3 == 2:
            parents = rng.integers(-1, len(lengths), sequences)
            lengths, _ = both.fork(lengths, parents)
            lengths = lengths.astype(np.int64)
        if turn % 4 == 3:
            both.compact()
    both.release()
    assert not both.plain.refs.any()


def test_pages_run_out(cuda):
    """Fewer pages than slots, a table that is too narrow, and forks without a page for their copy."""
    both = Both(cuda, 10, 32, 3, 6)
    assert both.reserve([0, 0, 0], [100, 7 * 32, 100]) == 4 + 6 + 1 + 4 - 10
    both.release(first=[0, 6, 0], last=[6, 6, 6])
    both.release()
    both.reserve([0, 0, 0], [100, 40, 100])
    # one row takes each parent over; two more want a copy of an unfinished page, and none is free
    assert both.plain.words().tolist() == [0]
    lengths, copies = both.fork([100, 40, 100], [0, 0, 2, 2])
    assert lengths.tolist() == [100, 96, 100, 96] and (copies.cpu() == -1).all()
    # the pages of the row without a child are free now
    assert both.plain.words().tolist() != [0]
    lengths, copies = both.fork(lengths, [0, 0, 0, 2])
    assert lengths.tolist() == [100, 100, 100, 100]


def test_numbers_that_make_no_sense(cuda):
    """Entries, parents, lengths, counts and ranges outside everything change nothing that they should not."""
    import torch

    both = Both(cuda, 40, 32, 4, 5)
    both.reserve([0, 0, 0, 0], [33, 64, 1, 160])
    both.table[0, 3] = both.expected[0, 3] = 4000
    both.table[1, 3] = both.expected[1, 3] = -7
    both.reserve([-5, 2 ** 30, 10 ** 6, 0], [-9, -1, -(2 ** 31), 0])
    both.release(first=[-100, 3, 9, 2], last=[-1, 2 ** 31 - 1, 10, 1])
    lengths, _ = both.fork([33, 64, -1, 160], [3, 0, 9, -2 ** 31, 3, 2 ** 31 - 1, 2])
    assert lengths.tolist() == [160, 33, 0, 0, 160, 0, 0]
    both.compact()
    both.release()
    # bits behind the last page are not pages
    both.pool.free[-1] = -1
    missing = both.paging.reserve(both.pool, both.table, torch.zeros(7, dtype=torch.int32, device=cuda),
                                  torch.full((7,), 160, dtype=torch.int32, device=cuda))
    held = both.table.cpu().numpy()
    assert int(missing) == 0 and held.min() >= -7 and len(set(held[held >= 0].tolist())) == (held >= 0).sum()


def test_slots_past_the_table(cuda):
    """Counts that reach far past the table: what is missing is counted, nothing is written there."""
    both = Both(cuda, 64, 32, 2, 3)
    assert both.reserve([0, 96], [32 * 10, 32 * 1000]) == 7 + 1000


def test_dropped_tokens_in_a_page_that_a_fork_holds(cuda):
    """The next fork gives each of those that end in it a page of its own, or none where there is none."""
    both = Both(cuda, 12, 32, 1, 4)
    both.reserve([0], [83])
    lengths, _ = both.fork([83], [0, 0, 0])  # two pages shared, three unfinished ones
    both.release(first=[3, 2, 2])
    lengths, copies = both.fork([83, 50, 50], [0, 1, 2])
    assert lengths.tolist() == [83, 50, 50] and (copies[:, 0] == int(both.expected[0, 1])).sum() == 2
    assert len(set(both.expected[:, 1].tolist())) == 3
    lengths, copies = both.fork(lengths, [2, 1, 0, 1])  # pages of their own move on
    assert (copies[:, 0] >= 0).sum() == 1
    both.release()
    assert not both.plain.refs.any()
    both = Both(cuda, 3, 32, 2, 4)
    both.reserve([0, 0], [64, 0])
    both.fork([64, 0], [0, 0])
    lengths, copies = both.fork([40, 41], [0, 1])  # one page is left for two
    assert lengths.tolist() == [40, 32] and (copies[:, 0] >= 0).sum() == 1


def test_smallest_pools_and_batches(cuda):
    """A pool of one page, tables without rows, forks to none and from none."""
    from ivonar_amd import attention

    both = Both(cuda, 1, 32, 1, 1)
    both.reserve([0], [5])
    assert both.compact().shape == (0, 2)
    lengths, copies = both.fork([5], [])
    assert lengths.shape == (0,) and copies.shape == (0, 2) and not both.plain.refs.any()
    assert both.reserve([], []) == 0
    both.release()
    both.compact()
    lengths, copies = both.fork([], [-1, 0])
    assert lengths.tolist() == [0, 0] and (copies.cpu() == -1).all()
    pages = attention.cache_pages(1, 1, 64, 32, cuda)
    both.paging.copy(pages, copies)
    both.paging.copy(pages, copies[:0])


@pytest.mark.parametrize("kv,dim,page,count", [(1, 64, 32, 40), (8, 128, 64, 60), (3, 256, 128, 9)])
def test_copies(cuda, kv, dim, page, count):
    """Forked and compacted sequences read back what they held, in every layer, and nothing else changes."""
    import torch
    from ivonar_amd import attention, paging

    rng = np.random.default_rng(dim)
    both = Both(cuda, count, page, 3, 8)
    layers = [attention.cache_pages(count, kv, dim, page, cuda) for _ in range(2)]
    for pages in layers:
        pages.copy_(torch.randint(0, 256, pages.shape, dtype=torch.uint8))
    lengths = np.array([page + 5, 2 * page, page // 2])
    both.reserve(np.zeros(3), lengths)
    parents = [0, 1, 0, 2, 2]

    def bytes_of(pages, row, length):
        return pages.cpu().numpy()[both.expected[row, :-(-int(length) // page)]]

    before = [[bytes_of(pages, p, lengths[p]) for p in parents] for pages in layers]
    whole = [pages.clone() for pages in layers]
    new_lengths, copies = both.fork(lengths, parents)
    assert new_lengths.tolist() == lengths[parents].tolist()
    for pages, old, kept in zip(layers, whole, before):
        paging.copy(pages, copies)
        for row, length in enumerate(new_lengths):
            assert np.array_equal(bytes_of(pages, row, length), kept[row])
        changed = (pages != old).flatten(1).any(1).nonzero().flatten().tolist()
        assert set(changed) <= set(copies[:, 1].tolist())
    both.release(last=[8, 0, 0, 0, 0])
    kept = [[bytes_of(pages, row, new_lengths[row]) for row in range(1, 5)] for pages in layers]
    copies = both.compact()
    for pages, rows in zip(layers, kept):
        paging.copy(pages, copies)
        for row, expected in zip(range(1, 5), rows):
            assert np.array_equal(bytes_of(pages, row, new_lengths[row]), expected)


def test_copy_lists(cuda):
    """Numbers outside the pages and copies onto themselves are skipped, wherever in the list they are."""
    import torch
    from ivonar_amd import paging

    pages = torch.randint(0, 256, (20, 2, 2, 34 * 64), dtype=torch.uint8, device=cuda)
    expected = pages.clone()
    paging.copy(pages, _ints(cuda, [[3, 4], [20, 5], [6, 20], [6, -1], [7, 7], [0, 19], [-1, 8], [9, 10]]))
    expected[4], expected[19], expected[10] = expected[3], expected[0], expected[9]
    assert torch.equal(pages, expected)
    paging.copy(pages, _ints(cuda, np.zeros((0, 2))))
    assert torch.equal(pages, expected)
    paging.copy(pages, _ints(cuda, [0, 17, 18]).unfold(0, 2, 1)[1:2].contiguous())  # on any address
    paging.copy(pages, torch.cat((_ints(cuda, [0]), _ints(cuda, [11, 12])))[1:].view(1, 2))
    expected[18], expected[12] = expected[17], expected[11]
    assert torch.equal(pages, expected)


def test_copies_past_32_bits(cuda):
    """Pages that lie more than 4 GiB into the cache, and more copies than blocks."""
    import torch
    from ivonar_amd import paging

    pages = torch.empty((70000, 8, 4, 34 * 64), dtype=torch.uint8, device=cuda)  # 4.9 GB
    pages.view(torch.int32)[:] = torch.arange(70000, dtype=torch.int32, device=cuda).view(-1, 1, 1, 1)
    copies = torch.stack((torch.arange(69000, 64000, -1), torch.arange(5000)), 1).to(torch.int32).to(cuda)
    paging.copy(pages, copies)
    held = pages.view(torch.int32)
    for part in (held[:, 0, 0, 0], held[:, 7, 3, -1]):
        assert torch.equal(part[:5000], torch.arange(69000, 64000, -1, device=cuda).int())
        assert torch.equal(part[5000:], torch.arange(5000, 70000, device=cuda).int())


def test_captured(cuda):
    """A decoding step's reservation and window release, and a fork into other tensors, replayed."""
    import torch
    from ivonar_amd import paging

    pool = paging.page_pool(300, 32, cuda)
    plain = _paging.Pool(300, 32)
    table = torch.full((6, 40), -1, dtype=torch.int32, device=cuda)
    expected = table.cpu().numpy()
    lengths = torch.zeros(6, dtype=torch.int32, device=cuda)
    counts = torch.full((6,), 25, dtype=torch.int32, device=cuda)
    parents = _ints(cuda, [0, 2, 2, 5, -1, 0])
    other, other_lengths = torch.empty_like(table), torch.empty_like(lengths)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        missing = paging.reserve(pool, table, lengths, counts)
        lengths.add_(counts)
        paging.release(pool, table, last=(lengths - 64).clamp_min(0) // 32)
        fork = paging.fork(pool, table, lengths, parents, out=(other, other_lengths))
        table.copy_(other)
        lengths.copy_(other_lengths)
    length = np.zeros(6, dtype=np.int64)
    for replay in range(5):
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert int(missing) == plain.reserve(expected, length, [25] * 6) == 0
        length = length + 25
        plain.release(expected, None, np.maximum(length - 64, 0) // 32)
        expected, length, copies, lacking = plain.fork(expected, length, [0, 2, 2, 5, -1, 0])
        length = length.astype(np.int64)
        assert np.array_equal(table.cpu().numpy(), expected) and np.array_equal(pool.refs.cpu().numpy(), plain.refs)
        assert np.array_equal(pool.free.cpu().numpy(), plain.words()) and int(fork.missing) == lacking
        assert np.array_equal(lengths.cpu().numpy(), length)
        assert fork.copies[:len(copies)].tolist() == [list(c) for c in copies]
        paging.page_pool(5, 32, cuda)  # the program's own work between replays


def test_refusals(cuda):
    import torch
    from ivonar_amd import attention, paging
    from ivonar_amd.runtime import KernelError

    for bad in ((0, 64), (-1, 64), (10, 48), (10, 16), ((1 << 27) + 1, 64)):
        with pytest.raises(KernelError):
            paging.page_pool(*bad, cuda)
    pool = paging.page_pool(40, 64, cuda)
    table, two = torch.full((2, 3), -1, dtype=torch.int32, device=cuda), _ints(cuda, [0, 0])
    calls = {"reserve": dict(table=table, lengths=two, counts=two), "release": dict(table=table, first=two, last=two),
             "fork": dict(table=table, lengths=two, parents=two), "compact": dict(table=table)}
    pools = (pool._replace(refs=pool.refs.long()), pool._replace(refs=pool.refs[:33]), pool._replace(free=pool.free[:1]),
             pool._replace(free=pool.free.cpu()), pool._replace(page_size=48), pool._replace(refs=pool.refs[:0]))
    for name, good in calls.items():
        call = getattr(paging, name)
        call(pool, **good)
        for bad in pools[:1] + pools[2:]:
            with pytest.raises(KernelError):
                call(bad, **good)
        for key, value in (("table", table.long()), ("table", table[0]), ("table", table[:, :2]), ("table", table.cpu()),
                           ("table", table[:, :0])):
            with pytest.raises(KernelError):
                call(pool, **{**good, key: value})
        for key in good:
            if key != "table":
                for value in (two.long(), two.cpu(), two[None]) + ((two[:1],) if key != "parents" else ()):
                    with pytest.raises(KernelError):
                        call(pool, **{**good, key: value})
    good = calls["fork"]
    for out in ((table, two.clone()), (table.clone(), two), (table[:1], two.clone()), (table.clone(), two[:1]),
                (table.clone().long(), two.clone())):
        with pytest.raises(KernelError):
            paging.fork(pool, **good, out=out)
    with pytest.raises(KernelError):
        wide = torch.full((8193, 1), -1, dtype=torch.int32, device=cuda)
        paging.fork(pool, wide, torch.zeros(8193, dtype=torch.int32, device=cuda), two)
    pages = attention.cache_pages(4, 1, 64, 32, cuda)
    for bad in ((pages.float(), _ints(cuda, [[0, 1]])), (pages[0], _ints(cuda, [[0, 1]])), (pages, two),
                (pages, _ints(cuda, [[0, 1]]).long()), (pages, _ints(cuda, [[0, 1, 2]])), (pages, _ints(cuda, [[0, 1]]).cpu()),
                (pages[:, :, :, :-8], _ints(cuda, [[0, 1]]))):
        with pytest.raises(KernelError):
            paging.copy(*bad)
    none = paging.fork(pool, table[:0], two[:0], two)
    assert (none.table == -1).all() and not none.lengths.any()
    gone = paging.fork(pool, none.table, none.lengths, two[:0])
    assert gone.table.shape == (0, 3) and gone.copies.shape == (0, 2) and int(gone.missing) == 0
