"""The 4-bit cache: rows written and read back against a plain 64-bit quantiser, value for value."""

from __future__ import annotations

import numpy as np
import pytest

import _attention as A

pytestmark = pytest.mark.gpu


def _table(cuda, table):
    import torch

    return torch.from_numpy(table).to(cuda)


def _ints(cuda, values):
    import torch

    return torch.tensor(values, dtype=torch.int32, device=cuda)


def _prefix(counts):
    return [0, *np.cumsum(counts).tolist()]


def _garbage(pages):
    """Arbitrary bytes, as in pages that held other sequences."""
    import torch

    pages.copy_(torch.randint(0, 256, pages.shape, dtype=torch.uint8))
    return pages


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("dim,heads,page", [(64, 3, 32), (128, 2, 64), (256, 1, 128), (128, 1, 32)])
def test_round_trip(cuda, rng, dtype, dim, heads, page):
    """Ragged rows (one sequence without any) at positions that start and end inside tiles and pages."""
    import torch
    from ivonar_amd import attention

    counts, past = [1, 0, 77, 33, 200], [5, 9, 0, 31, 63]
    pages_needed, table = A.place([p + c for p, c in zip(past, counts)], page, rng)
    pages = _garbage(attention.cache_pages(pages_needed, heads, dim, page, cuda))
    rows = sum(counts)
    k, v = (torch.randn(rows, heads, dim, device=cuda) * torch.logspace(-3, 3, rows, device=cuda)[:, None, None]
            for _ in range(2))
    k, v = k.to(getattr(torch, dtype)), v.to(getattr(torch, dtype))
    before = pages.clone()
    at = (_table(cuda, table), _ints(cuda, past), _ints(cuda, _prefix(counts)))
    attention.cache_write(pages, k, v, *at)
    for out in ("float32", "bfloat16", "float16"):
        got = attention.cache_read(pages, *at, rows, getattr(torch, out))
        for x, y in zip((k, v), got):
            expected = torch.from_numpy(A.stored(x.float().cpu().numpy())).to(getattr(torch, out))
            assert torch.equal(y.cpu(), expected), out
    # nothing else was touched: 17 bytes of 32 values for K and V each
    changed = int((pages != before).sum())
    assert changed <= rows * heads * dim * 34 // 32
    start = [max(0, p - 3) for p in past]  # another stretch: the same tokens where both have them
    longer = [c + p - s for c, p, s in zip(counts, past, start)]
    wide = attention.cache_read(pages, at[0], _ints(cuda, start), _ints(cuda, _prefix(longer)), sum(longer))
    for b, (count, more) in enumerate(zip(counts, longer)):
        begin, end = _prefix(counts)[b], _prefix(longer)[b + 1]
        for x, y in zip(got, wide):
            assert torch.equal(x[begin:begin + count].float(), y[end - count:end].to(x.dtype).float())


def test_edge_values(cuda):
    """Ties, zeros, the ends of the exponents' range, subnormals, and blocks with infinities and NaN."""
    import torch
    from ivonar_amd import attention

    rows = np.zeros((12, 1, 64), dtype=np.float32)
    rows[0, 0, :14] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -0.75, -1.25, -2.5, -5, -0.0]
    rows[1, 0, 0], rows[1, 0, 1] = 1.75, -1.7499999  # a block whose largest value moves the exponent up
    rows[1, 0, 32], rows[1, 0, 33] = 1.7499999, 0.3
    rows[2, 0, :3] = [3.4e38, -3.3e38, 1e30]
    rows[3, 0, :3] = [1e-38, 1e-45, -1e-40]
    rows[4, 0, :3] = [2.0 ** -98, 2.0 ** -99, 2.0 ** -101]
    rows[5, 0, :2] = [np.inf, 1.0]
    rows[5, 0, 40] = 2.0
    rows[6, 0, 63] = np.nan
    rows[7, 0, 3] = -np.inf
    rows[8] = np.float32(7.0)
    rows[9, 0, ::2] = np.linspace(-7, 7, 32)
    x = torch.from_numpy(rows).to(cuda)
    pages = attention.cache_pages(2, 1, 64, 32, cuda)
    at = (_ints(cuda, [[1]]), _ints(cuda, [0]), _ints(cuda, [0, 12]))
    attention.cache_write(pages, x, x, *at)
    for got in attention.cache_read(pages, *at, 12):
        assert np.array_equal(got.cpu().numpy().astype(np.float64), A.stored(rows), equal_nan=True)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_strided_rows(cuda, rng, dtype):
    """k and v as parts of one projection's output, off every alignment, and heads apart from tokens."""
    import torch
    from ivonar_amd import attention

    heads, dim, rows = 2, 64, 70
    pages_needed, table = A.place([rows], 64, rng)
    at = (_table(cuda, table), _ints(cuda, [0]), _ints(cuda, [0, rows]))
    for offset in (0, 1, 4, 8):
        fused = torch.randn(rows, 4 * heads * dim + 24, device=cuda).to(getattr(torch, dtype))
        k = fused[:, offset:offset + heads * dim].unflatten(1, (heads, dim))
        v = fused[:, 256 + offset:256 + offset + heads * dim].unflatten(1, (heads, dim))
        pages = attention.cache_pages(pages_needed, heads, dim, 64, cuda)
        attention.cache_write(pages, k, v, *at)
        for x, y in zip((k, v), attention.cache_read(pages, *at, rows)):
            assert np.array_equal(y.cpu().numpy(), A.stored(x.float().cpu().numpy())), offset
    k, v = (torch.randn(heads, rows, dim, device=cuda).transpose(0, 1) for _ in range(2))
    attention.cache_write(pages, k, v, *at)
    for x, y in zip((k, v), attention.cache_read(pages, *at, rows)):
        assert np.array_equal(y.cpu().numpy(), A.stored(x.cpu().numpy()))


def test_rows_without_a_place(cuda):
    """Rows of no sequence, positions without a page and negative positions are not written, and read as zero."""
    import torch
    from ivonar_amd import attention

    pages = attention.cache_pages(3, 1, 64, 32, cuda)
    table = _ints(cuda, [[0, -1, 1], [3, 2, -7], [2, 2, 2]])
    x = torch.randn(120, 1, 64, device=cuda)
    offsets = _ints(cuda, [0, 70, 100, 110])  # 10 rows of no sequence at the end
    past = _ints(cuda, [10, 20, -5])
    attention.cache_write(pages, x, x, table, past, offsets)
    expected = A.stored(x.cpu().numpy())
    got = attention.cache_read(pages, table, past, offsets, 120)[0].cpu().numpy()
    zero = np.zeros((1, 64))
    for row in range(120):
        if row < 70:
            there = not 32 <= 10 + row < 64
        elif row < 100:
            there = 32 <= 20 + row - 70
        else:
            there = False
        assert np.array_equal(got[row], expected[row] if there else zero), row
    # a page table narrower than the sequence: rows past it have no place
    pages.zero_()
    attention.cache_write(pages, x, x, _ints(cuda, [[2]]), _ints(cuda, [0]), _ints(cuda, [0, 120]))
    assert int(pages[:2].max()) == 0
    got = attention.cache_read(pages, _ints(cuda, [[2]]), None, _ints(cuda, [0, 120]), 120)[1].cpu().numpy()
    assert np.array_equal(got[:32], expected[:32]) and not got[32:].any()


@pytest.mark.parametrize("sequences", [1, 63, 64, 65, 200])
def test_many_sequences(cuda, rng, sequences):
    """One row each without offsets, and rows of many short sequences, some of them empty."""
    import torch
    from ivonar_amd import attention

    past = rng.integers(0, 100, sequences).tolist()
    for counts in ([1] * sequences, [int(c) for c in rng.integers(0, 4, sequences)]):
        pages_needed, table = A.place([p + c for p, c in zip(past, counts)], 32, rng)
        pages = _garbage(attention.cache_pages(pages_needed, 2, 128, 32, cuda))
        x = torch.randn(sum(counts), 2, 128, device=cuda)
        y = torch.randn(sum(counts), 2, 128, device=cuda)
        offsets = None if counts == [1] * sequences else _ints(cuda, _prefix(counts))
        at = (_table(cuda, table), _ints(cuda, past), offsets)
        attention.cache_write(pages, x, y, *at)
        got = attention.cache_read(pages, *at, sum(counts))
        for a, b in zip((x, y), got):
            assert np.array_equal(b.cpu().numpy(), A.stored(a.cpu().numpy()))


def test_addresses_past_32_bits(cuda):
    """Pages that lie more than 4 GiB into the cache."""
    import torch
    from ivonar_amd import attention

    pages = torch.empty((70000, 8, 4, 34 * 64), dtype=torch.uint8, device=cuda)  # 4.9 GB
    last = pages.shape[0] - 1
    table = _ints(cuda, [[last, 0], [1, last - 1]])
    x, y = (torch.randn(300, 8, 64, device=cuda) for _ in range(2))
    at = (table, _ints(cuda, [100, 0]), _ints(cuda, [0, 150, 300]))
    attention.cache_write(pages, x, y, *at)
    for a, b in zip((x, y), attention.cache_read(pages, *at, 300)):
        assert np.array_equal(b[:150].cpu().numpy(), A.stored(a[:150].cpu().numpy()))
        assert np.array_equal(b[150:].cpu().numpy(), A.stored(a[150:].cpu().numpy()))
    q = torch.randn(2, 8, 64, device=cuda)
    out = attention.cache_attention(q, pages, table, _ints(cuda, [250, 150]))
    kept = [A.stored(a.cpu().numpy()) for a in (x, y)]
    zeros = np.zeros((100, 8, 64))
    pages[last].zero_()
    attention.cache_write(pages, x, y, *at)
    out = attention.cache_attention(q, pages, table, _ints(cuda, [250, 150])).cpu().numpy()
    for b, (rows, before) in enumerate(((slice(0, 150), zeros), (slice(150, 300), zeros[:0]))):
        k, v = (np.concatenate((before, side[rows])) for side in kept)
        result = A.attend(q[b:b + 1].cpu().numpy(), k, v, k.shape[0] - 1)
        A.check(out[b:b + 1], *result, "float32", k.shape[0], 64)


def test_refusals(cuda):
    import torch
    from ivonar_amd import attention
    from ivonar_amd.runtime import KernelError, library

    for bad in ((0, 1, 64, 64), (1, 0, 64, 64), (1, 1, 80, 64), (1, 1, 64, 48), (1, 1, 64, 16)):
        with pytest.raises(KernelError):
            attention.cache_pages(*bad, cuda)
    pages = attention.cache_pages(2, 2, 64, 64, cuda)
    table, zero, offsets = _ints(cuda, [[0, 1]]), _ints(cuda, [0]), _ints(cuda, [0, 4])
    x = torch.zeros(4, 2, 64, device=cuda)
    good = dict(pages=pages, k=x, v=x, table=table, past=zero, offsets=offsets)
    attention.cache_write(**good)
    for name, value in (("k", x[:3]), ("k", x[:, :1]), ("k", x[..., :32]), ("k", x.double()), ("k", x.half()),
                        ("v", x.flatten(1)), ("k", x.transpose(1, 2).contiguous().transpose(1, 2)), ("k", x.cpu()),
                        ("pages", pages.float()), ("pages", pages[..., :-2]), ("pages", pages[:, :1]),
                        ("table", table.long()), ("table", table[0]), ("table", table.cpu()),
                        ("past", _ints(cuda, [0, 0])), ("past", zero.long()), ("offsets", zero), ("offsets", None),
                        ("offsets", offsets.cpu())):
        with pytest.raises(KernelError):
            attention.cache_write(**{**good, name: value})
    with pytest.raises(KernelError):
        attention.cache_read(pages, table, zero, offsets, 4, torch.float64)
    with pytest.raises(KernelError):
        attention.cache_read(pages, table, zero, offsets, -1)
    k, v = attention.cache_read(pages, table, zero, _ints(cuda, [0, 0]), 0)
    assert k.shape == v.shape == (0, 2, 64)
    # the C entry refuses what the Python side would not let through, without a launch
    lib, p = library(), pages.data_ptr()
    tail = (table.data_ptr(), 2, zero.data_ptr(), offsets.data_ptr(), 1)
    head = (0, x.data_ptr(), x.data_ptr(), 0, 128, 64, 128, 64, 4)
    assert lib.ivonar_cache_write(*head, p, 2, 2, 2, 64, *tail) == 0
    for change in ((p + 1, 2, 2, 2, 64), (None, 2, 2, 2, 64), (p, 0, 2, 2, 64), (p, 2, 2, 3, 64), (p, 2, 2, 2, 96),
                   (p, 2, -1, 2, 64)):
        assert lib.ivonar_cache_write(*head, *change, *tail) != 0
    assert lib.ivonar_cache_write(0, x.data_ptr(), x.data_ptr(), 3, 128, 64, 128, 64, 4, p, 2, 2, 2, 64, *tail) != 0
    assert lib.ivonar_cache_write(*head, p, 2, 2, 2, 64, table.data_ptr(), 1 << 26, *tail[2:]) != 0
