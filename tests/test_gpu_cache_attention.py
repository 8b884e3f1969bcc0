"""Attention over the 4-bit cache against 64-bit attention over the values that the cache holds."""

from __future__ import annotations

import numpy as np
import pytest

import _attention as A

pytestmark = pytest.mark.gpu


def _ints(cuda, values):
    import torch

    return torch.tensor(values, dtype=torch.int32, device=cuda)


class Case:
    """A cache filled with random keys and values of sequences of these lengths, unwritten bytes arbitrary."""

    def __init__(self, cuda, rng, lengths, kv_heads, dim, page=64, spread=1.0):
        import torch
        from ivonar_amd import attention

        self.lengths, self.kv_heads, self.dim, self.cuda = lengths, kv_heads, dim, cuda
        count, table = A.place(lengths, page, rng)
        self.pages = attention.cache_pages(count, kv_heads, dim, page, cuda)
        self.pages.copy_(torch.randint(0, 256, self.pages.shape, dtype=torch.uint8))
        self.table = torch.from_numpy(table).to(cuda)
        rows = [(rng.standard_normal((n, kv_heads, dim)) * spread).astype(np.float32) for n in lengths for _ in "kv"]
        self.k, self.v = rows[0::2], rows[1::2]
        offsets = _ints(cuda, [0, *np.cumsum(lengths).tolist()])
        if sum(lengths):
            attention.cache_write(self.pages, torch.from_numpy(np.concatenate(self.k)).to(cuda),
                                  torch.from_numpy(np.concatenate(self.v)).to(cuda), self.table,
                                  _ints(cuda, [0] * len(lengths)), offsets)
        self.k, self.v = [A.stored(x) for x in self.k], [A.stored(x) for x in self.v]

    def run(self, rng, heads, dtype, queries=None, check=True, **options):
        """queries: rows per sequence, None for one each without offsets."""
        import torch
        from ivonar_amd import attention

        counts = [1] * len(self.lengths) if queries is None else queries
        q = torch.from_numpy(rng.standard_normal((sum(counts), heads, self.dim)).astype(np.float32)).to(self.cuda)
        q = q.to(getattr(torch, dtype))
        starts = [0, *np.cumsum(counts).tolist()]
        offsets = None if queries is None else _ints(self.cuda, starts)
        out = attention.cache_attention(q, self.pages, self.table, _ints(self.cuda, self.lengths), offsets, **options)
        assert out.dtype == q.dtype and out.shape == q.shape
        options = {name: options[name] for name in ("window", "sinks", "scale") if name in options}
        if check:
            got, rows = out.float().cpu().numpy(), q.float().cpu().numpy()
            for b, (length, count) in enumerate(zip(self.lengths, counts)):
                part = slice(starts[b], starts[b + 1])
                result = A.attend(rows[part], self.k[b], self.v[b], length - count, **options)
                A.check(got[part], *result, dtype, length, self.dim, f"sequence {b}")
        return q, out


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("dim,kv_heads,heads", [(64, 2, 2), (64, 1, 8), (128, 2, 6), (128, 1, 20), (256, 2, 4)])
def test_single_tokens(cuda, rng, dtype, dim, kv_heads, heads):
    """Lengths of zero, one, and around the ends of tiles and pages."""
    case = Case(cuda, rng, [1, 0, 31, 32, 33, 64, 65, 127, 300, 700], kv_heads, dim)
    case.run(rng, heads, dtype)
    case.run(rng, heads, dtype, queries=[1] * 10)


@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 1), (32, 4), (33, 40), (64, 64), (200, 33), (1000, 4), (7, 600)])
def test_window_and_sinks(cuda, rng, window, sinks):
    case = Case(cuda, rng, [1, 6, 64, 97, 260, 500], 2, 64, page=32)
    case.run(rng, 4, "float32", window=window, sinks=sinks)
    case.run(rng, 4, "bfloat16", queries=[1, 6, 20, 40, 3, 70], window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("dim,heads", [(64, 2), (64, 14), (128, 8), (256, 4)])
def test_several_tokens(cuda, rng, dtype, dim, heads):
    """Chunks of any length, an empty one and a whole sequence among them."""
    case = Case(cuda, rng, [90, 1, 64, 130, 33], 2, dim)
    case.run(rng, heads, dtype, queries=[17, 1, 64, 0, 5])
    case.run(rng, heads, dtype, queries=[90, 0, 1, 129, 33])


@pytest.mark.parametrize("length,max_length", [(5000, 5000), (5000, 40), (5000, 1 << 20), (700, 1 << 20)])
def test_shared_axis(cuda, rng, length, max_length):
    """One row per head and many keys, split over blocks, whatever the length that the caller announces."""
    case = Case(cuda, rng, [length, 100], 1, 128, page=128)
    case.run(rng, 4, "float32", max_length=max_length)
    case.run(rng, 4, "bfloat16", queries=[3, 2], max_length=max_length, window=2000, sinks=70)


@pytest.mark.parametrize("dim,heads,dtype", [(64, 4, "bfloat16"), (64, 3, "float32"), (128, 4, "float16"),
                                             (256, 2, "bfloat16")])
@pytest.mark.parametrize("max_length", [600, 1 << 16])
def test_many_sequences(cuda, rng, dim, heads, dtype, max_length):
    """More sequences than lanes, most short and one long: blocks that end one row tile, take whole ones and begin
    another, or one block for each, by the length that the caller announces."""
    lengths = [int(n) for n in rng.integers(0, 500, 150)]
    lengths[3], lengths[70], lengths[149] = 2600, 0, 33
    case = Case(cuda, rng, lengths, 1, dim, page=32)
    case.run(rng, heads, dtype, max_length=max_length)
    queries = [int(n) for n in rng.integers(0, 4, 150)]
    queries[3], queries[60] = 40, 0
    case.run(rng, heads, dtype, queries=queries, max_length=max_length)


@pytest.mark.parametrize("rows", [8, 12, 30])
def test_row_tiles_that_share_blocks(cuda, rng, rows):
    """Row tiles of 8, 16 and 32 rows of few sequences, whose keys begin and end inside blocks."""
    case = Case(cuda, rng, [1200, 900, 2100], 2, 64)
    case.run(rng, 2, "bfloat16", queries=[rows, rows - 5, rows + 3], max_length=4000)
    case.run(rng, 2, "float32", queries=[rows, 0, rows + 9], max_length=4000, window=700, sinks=40)


@pytest.mark.parametrize("dim,heads,dtype", [(64, 2, "float32"), (128, 2, "bfloat16"), (256, 1, "float16")])
def test_long_chunks(cuda, rng, dim, heads, dtype):
    """Many row tiles, each of whose keys are split at equal lengths."""
    case = Case(cuda, rng, [3000, 700], 1, dim)
    case.run(rng, heads, dtype, queries=[611, 10])
    case.run(rng, heads, dtype, queries=[400, 300], window=1500, sinks=5)


def test_more_queries_than_tokens(cuda, rng):
    """Rows before the sequence's first position see nothing and are zero."""
    case = Case(cuda, rng, [3, 0], 1, 64)
    _, out = case.run(rng, 2, "float32", queries=[5, 4])
    got = out.cpu().numpy()
    assert not got[:2].any() and not got[5:].any() and got[2:5].any(-1).all()


def test_rows_of_no_sequence(cuda, rng):
    import torch
    from ivonar_amd import attention

    case = Case(cuda, rng, [40, 70], 1, 64)
    q = torch.randn(30, 3, 64, device=cuda)
    lengths = _ints(cuda, case.lengths)
    out = torch.full_like(q, float("nan"))
    attention.cache_attention(q, case.pages, case.table, lengths, _ints(cuda, [2, 9, 20]), out=out)
    got = out.cpu().numpy()
    assert not got[:2].any() and not got[20:].any()
    for b, part in enumerate((slice(2, 9), slice(9, 20))):
        count = part.stop - part.start
        result = A.attend(q[part].cpu().numpy(), case.k[b], case.v[b], case.lengths[b] - count)
        A.check(got[part], *result, "float32", 70, 64)


def test_pages_that_are_not_there(cuda, rng):
    """Entries outside the pages are not seen: pages before a window may be gone, and a row may see none at all."""
    import torch
    from ivonar_amd import attention

    case = Case(cuda, rng, [300, 300, 60], 2, 128, page=32)
    table = case.table.clone()
    table[0, 2:5] = -1
    table[1, 1:8] = 1 << 30
    table[2, :] = -3
    q = torch.randn(3, 4, 128, device=cuda)
    lengths = _ints(cuda, case.lengths)
    got = attention.cache_attention(q, case.pages, table, lengths).cpu().numpy()
    key = np.arange(300)
    for b, missing in enumerate(((key >= 64) & (key < 160), (key >= 32) & (key < 256), key >= 0)):
        length = case.lengths[b]
        result = A.attend(q[b:b + 1].cpu().numpy(), case.k[b], case.v[b], length - 1, missing=missing[:length])
        A.check(got[b:b + 1], *result, "float32", length, 128)
    assert not got[2].any()
    whole = attention.cache_attention(q, case.pages, case.table, lengths, window=40, sinks=20)
    kept = attention.cache_attention(q[:2], case.pages, table[:2], lengths[:2], window=40, sinks=20)
    assert torch.equal(whole[:2], kept)
    # a length past what the table can hold ends there
    narrow = case.table[:1, :2].contiguous()
    got = attention.cache_attention(q[:1], case.pages, narrow, _ints(cuda, [300])).cpu().numpy()
    result = A.attend(q[:1].cpu().numpy(), case.k[0][:64], case.v[0][:64], 63)
    A.check(got, *result, "float32", 64, 128)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_no_number_stays_where_it_is_seen(cuda, rng, dim):
    """A block without a number reaches the rows that see its token, in its 32 dims, and no others."""
    import torch
    from ivonar_amd import attention

    case = Case(cuda, rng, [90], 1, dim)
    bad_key, bad_value = np.zeros((1, 1, dim), np.float32), np.zeros((1, 1, dim), np.float32)
    bad_value[0, 0, 40] = np.inf
    for token in (70, 75):  # token 70: a value; 75: a key and a value
        if token == 75:
            bad_key[0, 0, 0] = np.nan
        attention.cache_write(case.pages, torch.from_numpy(bad_key).to(cuda), torch.from_numpy(bad_value).to(cuda),
                              case.table, _ints(cuda, [token]))
        case.k[0][token], case.v[0][token] = A.stored(bad_key)[0], A.stored(bad_value)[0]
    for dtype in ("float32", "bfloat16"):
        q, out = case.run(rng, 2, dtype, queries=[30], check=False)  # positions 60 .. 89
        got, rows = out.float().cpu().numpy(), q.float().cpu().numpy()
        for i in range(30):
            missing = np.zeros(90, bool)
            missing[[70, 75]] = True
            expected, spread, size = A.attend(rows[i:i + 1], case.k[0], case.v[0], 60 + i, missing=missing)
            if 60 + i < 70:
                A.check(got[i:i + 1], expected, spread, size, dtype, 90, dim, f"row {i}")
            elif 60 + i < 75:
                assert np.isnan(got[i, :, 32:64]).all()
                assert np.isfinite(got[i, :, :32]).all() and np.isfinite(got[i, :, 64:]).all()
            else:
                assert np.isnan(got[i]).all()
        _, out = case.run(rng, 2, dtype, queries=[1], check=False, window=10)  # 80 .. 89: past both
        assert torch.isfinite(out.float()).all()


def test_large_logits(cuda, rng):
    """Logits far apart, in the thousands, whose running maximum rises over and over."""
    case = Case(cuda, rng, [400], 1, 64)
    import torch
    from ivonar_amd import attention

    k = np.zeros((400, 1, 64), np.float32)
    k[:, 0, 0] = 6.0 * 2.0 ** (np.arange(400) % 9)
    k[::2] *= -1
    v = rng.standard_normal((400, 1, 64)).astype(np.float32)
    attention.cache_write(case.pages, torch.from_numpy(k).to(cuda), torch.from_numpy(v).to(cuda), case.table,
                          _ints(cuda, [0]), _ints(cuda, [0, 400]))
    case.k[0], case.v[0] = A.stored(k), A.stored(v)
    case.run(rng, 3, "float32")
    case.run(rng, 3, "float32", queries=[50], scale=4.0)


def test_strided_queries_and_output(cuda, rng):
    import torch
    from ivonar_amd import attention

    case = Case(cuda, rng, [50, 80], 2, 64)
    lengths = _ints(cuda, case.lengths)
    for dtype in (torch.float32, torch.bfloat16):
        fused = torch.randn(2, 4 * 64 * 2 + 3, device=cuda).to(dtype)
        for offset in (0, 1, 2):
            q = fused[:, offset:offset + 256].unflatten(1, (4, 64))
            expected = attention.cache_attention(q.contiguous(), case.pages, case.table, lengths)
            assert torch.equal(attention.cache_attention(q, case.pages, case.table, lengths), expected)
        q = torch.randn(4, 2, 64, device=cuda).to(dtype).transpose(0, 1)
        expected = attention.cache_attention(q.contiguous(), case.pages, case.table, lengths)
        out = torch.empty(2, 4, 64, dtype=dtype, device=cuda)
        assert attention.cache_attention(q, case.pages, case.table, lengths, out=out) is out
        assert torch.equal(out, expected)


def test_same_bits_every_time_and_in_a_graph(cuda, rng):
    """Results do not depend on the order in which blocks end; a captured step follows its buffers."""
    import torch
    from ivonar_amd import attention

    case = Case(cuda, rng, [3000, 2000, 40], 2, 128)
    q = torch.randn(3, 8, 128, device=cuda).bfloat16()
    k, v = (torch.randn(3, 2, 128, device=cuda) for _ in range(2))
    past = _ints(cuda, [2990, 1999, 39])
    lengths = torch.empty_like(past)
    out = torch.empty_like(q)

    def step():
        attention.cache_write(case.pages, k, v, case.table, past)
        lengths.copy_(past + 1)
        attention.cache_attention(q, case.pages, case.table, lengths, out=out)

    step()
    first = out.clone()
    for _ in range(5):
        step()
        assert torch.equal(out, first)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for turn in range(4):
        past.add_(-turn)
        k.normal_()
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        step()
        torch.cuda.synchronize()
        assert torch.equal(out, replayed), turn


def test_on_two_streams(cuda, rng):
    import torch
    from ivonar_amd import attention

    case = Case(cuda, rng, [4000], 2, 128)
    lengths = _ints(cuda, [4000])
    qs = [torch.randn(1, 8, 128, device=cuda) for _ in range(2)]
    expected = [attention.cache_attention(q, case.pages, case.table, lengths) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    for _ in range(10):
        results = []
        for stream, q in zip(streams, qs):
            with torch.cuda.stream(stream):
                results.append(attention.cache_attention(q, case.pages, case.table, lengths))
        torch.cuda.synchronize()
        for a, b in zip(results, expected):
            assert torch.equal(a, b)


def test_refusals(cuda, rng):
    import torch
    from ivonar_amd import attention
    from ivonar_amd.runtime import KernelError, library

    case = Case(cuda, rng, [50], 2, 64)
    q, lengths = torch.zeros(1, 4, 64, device=cuda), _ints(cuda, [50])
    good = dict(q=q, pages=case.pages, table=case.table, lengths=lengths)
    attention.cache_attention(**good)
    for name, value in (("q", q[:, :3]), ("q", q[..., :32]), ("q", q.double()), ("q", q.cpu()), ("q", q[0]),
                        ("q", torch.zeros(2, 4, 64, device=cuda)), ("q", q[:, :0]), ("lengths", lengths.long()),
                        ("lengths", _ints(cuda, [1, 2])), ("offsets", _ints(cuda, [0])), ("window", -1), ("sinks", -1),
                        ("scale", 0.0), ("scale", float("nan")), ("scale", float("inf")), ("scale", -1.0),
                        ("out", q.half()), ("out", torch.zeros(1, 4, 128, device=cuda)[..., ::2]),
                        ("pages", case.pages.int()), ("table", case.table.float())):
        with pytest.raises(KernelError):
            attention.cache_attention(**{**good, name: value})
    empty = attention.cache_attention(q[:0], case.pages, case.table, lengths, _ints(cuda, [0, 0]))
    assert empty.shape == (0, 4, 64)
    # no sequences at all: every row is one of no sequence
    none = attention.cache_attention(q, case.pages, case.table[:0], lengths[:0], _ints(cuda, [0]))
    assert not none.any()
    lib = library()
    assert lib.ivonar_cache_attention_work(0, 4, 3, 64, None, 1, 1, 0, 0, 50) == -1
    need = lib.ivonar_cache_attention_work(0, 4, 2, 64, None, 1, 1, 0, 0, 1 << 20)
    assert need > 0

    def call(work, size, scale=0.125, window=0):
        return lib.ivonar_cache_attention(0, q.data_ptr(), 0, 256, 64, 4, 1, case.pages.data_ptr(),
                                          case.pages.shape[0], 2, 2, 64, case.table.data_ptr(), case.table.shape[1],
                                          lengths.data_ptr(), None, 1, window, 0, scale, 1 << 20, q.data_ptr(), work,
                                          size)

    work = torch.empty(need, dtype=torch.uint8, device=cuda)
    assert call(work.data_ptr(), need) == 0
    for bad in ((None, need), (work.data_ptr(), need - 1), (work.data_ptr() + 4, need), (work.data_ptr(), need, -1.0),
                (work.data_ptr(), need, 0.1, -1)):
        assert call(*bad) != 0


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_logits_past_the_integers(cuda, rng, dtype, dim):
    """Logits so large that fp32 holds them in steps of far more than one: the largest takes all the weight, and rows
    next to such a row come out as they do without it."""
    import torch
    from ivonar_amd import attention

    case = Case(cuda, rng, [400], 1, dim)
    k = np.zeros((400, 1, dim), np.float32)
    k[:, 0, 0] = rng.choice([0.0, 0.5, 1.0, -0.5], 400)
    for token, value in ((5, 1.5), (130, 4.0), (360, 6.0), (381, 8.0), (60, -1.0), (200, -6.0), (370, -12.0)):
        k[token] = value
    v = rng.standard_normal((400, 1, dim)).astype(np.float32)
    attention.cache_write(case.pages, torch.from_numpy(k).to(cuda), torch.from_numpy(v).to(cuda), case.table,
                          _ints(cuda, [0]), _ints(cuda, [0, 400]))
    key, value = A.stored(k)[:, 0, 0], A.stored(v)[:, 0]
    lengths = _ints(cuda, [400])
    for count in (1, 3, 8, 50):  # row tiles of every size
        q = torch.zeros(count, 2, dim, device=cuda, dtype=getattr(torch, dtype))
        q[:, 0, 0], q[:, 1, 0] = 2.0 ** 15, -2.0 ** 15
        offsets = _ints(cuda, [0, count])
        for scale in (2.0 ** 10, 2.0 ** 16, 2.0 ** 30):  # logits from 2^25 to 2^49
            out = attention.cache_attention(q, case.pages, case.table, lengths, offsets, scale=scale)
            out = out.double().cpu().numpy()
            for i in range(count):
                last = 400 - count + i
                for head, best in enumerate((key[:last + 1].argmax(), key[:last + 1].argmin())):
                    expected = torch.from_numpy(value[best]).to(q.dtype).double().numpy()
                    assert np.array_equal(out[i, head], expected), (count, scale, i, head)
        q = torch.randn(count, 2, dim, device=cuda).mul_(2.0 ** -10).to(q.dtype)
        q[::2, 1] = 0
        q[::2, 1, 0] = 2.0 ** 15
        out = attention.cache_attention(q, case.pages, case.table, lengths, offsets, scale=2.0 ** 10)
        q[::2, 1] = 0
        without = attention.cache_attention(q, case.pages, case.table, lengths, offsets, scale=2.0 ** 10)
        assert torch.equal(out[:, 0], without[:, 0]) and torch.equal(out[1::2], without[1::2])


@pytest.mark.parametrize("length,window,sinks", [(80, 0, 0), (80, 20, 3), (65, 1, 0), (5000, 64, 0), (5000, 64, 70),
                                                 (2 ** 31 - 1, 2 ** 30, 5), (2 ** 31 - 1, 0, 0)])
def test_lengths_past_the_table(cuda, rng, length, window, sinks):
    """Positions past the table have no page: the rows keep their positions, and see what the table holds of them."""
    import torch
    from ivonar_amd import attention

    case = Case(cuda, rng, [2048], 2, 64, page=32)
    for width in (2, 64):
        table = case.table[:, :width].contiguous()
        keys = 32 * width
        for count in (1, 5, 40):
            q = torch.randn(count, 4, 64, device=cuda)
            out = attention.cache_attention(q, case.pages, table, _ints(cuda, [length]), _ints(cuda, [0, count]), window,
                                            sinks).cpu().numpy()
            seen = min(keys, length)
            result = A.attend(q.cpu().numpy(), case.k[0][:seen], case.v[0][:seen], length - count, window, sinks)
            A.check(out, *result, "float32", keys, 64, f"{count} rows over {keys} tokens")


def test_misaligned_tensors_are_named(cuda, rng):
    import torch
    from ivonar_amd import attention
    from ivonar_amd.runtime import KernelError

    case = Case(cuda, rng, [50], 2, 64)
    q, lengths = torch.zeros(1, 4, 64, device=cuda), _ints(cuda, [50])
    out = torch.empty(4 * 64 + 1, device=cuda)[1:].view(1, 4, 64)
    with pytest.raises(KernelError, match="out .*16 bytes"):
        attention.cache_attention(q, case.pages, case.table, lengths, out=out)
    pages = torch.zeros(case.pages.numel() + 8, dtype=torch.uint8, device=cuda)[8:].view(case.pages.shape)
    kv = torch.zeros(1, 2, 64, device=cuda)
    for call in (lambda: attention.cache_attention(q, pages, case.table, lengths),
                 lambda: attention.cache_write(pages, kv, kv, case.table, lengths),
                 lambda: attention.cache_read(pages, case.table, lengths, None, 1)):
        with pytest.raises(KernelError, match="pages .*16 bytes"):
            call()


# The kernel rounds a weight to two bf16 terms for float16 and bfloat16 rows, and to three for float32 ones.
WEIGHT = {"float32": 2.0 ** -24, "float16": 2.0 ** -17, "bfloat16": 2.0 ** -17}


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("count", [1, 3, 8, 40])
def test_every_term_of_the_weights(cuda, dtype, dim, count):
    """Two thirds of the keys have a weight between two bfloat16 numbers, and values that nearly cancel those of the
    others: the results are much smaller than the values, so that their own rounding does not hide the weights'."""
    import torch
    from ivonar_amd import attention

    length = 300
    k, v, scale = A.cancelling(length, dim)
    pages = attention.cache_pages(8, 1, dim, 64, cuda)
    table = torch.arange(8, dtype=torch.int32, device=cuda).reshape(1, 8)
    attention.cache_write(pages, torch.from_numpy(k).to(cuda), torch.from_numpy(v).to(cuda), table, _ints(cuda, [0]),
                          _ints(cuda, [0, length]))
    assert np.array_equal(A.stored(k), k) and np.array_equal(A.stored(v), v)
    q = torch.zeros(count, 2, dim, device=cuda, dtype=getattr(torch, dtype))
    q[..., 0] = 1
    out = attention.cache_attention(q, pages, table, _ints(cuda, [length]), _ints(cuda, [0, count]), scale=scale)
    result = A.attend(q.float().cpu().numpy(), k, v, length - count, scale=scale)
    A.check(out.float().cpu().numpy(), *result, dtype, length, dim, weight_unit=WEIGHT[dtype])


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("count", [30, 4])
def test_no_number_with_half_queries(cuda, rng, dim, count):
    """As above for float16 queries, in row tiles of both kinds."""
    import torch
    from ivonar_amd import attention

    case = Case(cuda, rng, [90], 1, dim)
    key, value = np.zeros((1, 1, dim), np.float32), np.zeros((1, 1, dim), np.float32)
    value[0, 0, 40] = -np.inf
    attention.cache_write(case.pages, torch.from_numpy(key).to(cuda), torch.from_numpy(value).to(cuda), case.table,
                          _ints(cuda, [70]))
    key[0, 0, 0] = np.nan
    attention.cache_write(case.pages, torch.from_numpy(key).to(cuda), torch.zeros_like(torch.from_numpy(value)).to(cuda),
                          case.table, _ints(cuda, [88]))
    case.k[0][70], case.v[0][88] = 0, 0
    missing = np.zeros(90, bool)
    missing[[70, 88]] = True
    q, out = case.run(rng, 2, "float16", queries=[count], check=False)
    got, rows = out.float().cpu().numpy(), q.float().cpu().numpy()
    for i in range(count):
        position = 90 - count + i
        if position >= 88:
            assert np.isnan(got[i]).all()
        elif position >= 70:
            assert np.isnan(got[i, :, 32:64]).all()
            assert np.isfinite(got[i, :, :32]).all() and np.isfinite(got[i, :, 64:]).all()
        else:
            result = A.attend(rows[i:i + 1], case.k[0], case.v[0], position, missing=missing)
            A.check(got[i:i + 1], *result, "float16", 90, dim, f"row {i}")


def test_results_past_2_to_31_elements(cuda):
    import torch
    from ivonar_amd import attention

    rows, heads, dim = 131200, 64, 256
    pages = attention.cache_pages(2, 1, dim, 32, cuda)
    table = torch.arange(rows, device=cuda).remainder_(2).to(torch.int32).unsqueeze(1)
    v = torch.tensor([6.0, -3.0], device=cuda).reshape(2, 1, 1).expand(2, 1, dim).contiguous()
    attention.cache_write(pages, v, v, table[:2].contiguous(), _ints(cuda, [0, 0]))
    q = torch.zeros(rows, heads, dim, dtype=torch.bfloat16, device=cuda)
    out = attention.cache_attention(q, pages, table, torch.ones(rows, dtype=torch.int32, device=cuda))
    expected = v.bfloat16()
    for start in range(0, rows, 8200):
        assert torch.equal(out[start:start + 8200], expected.repeat(4100, heads, 1))
