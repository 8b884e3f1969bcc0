"""Norm and rotation of query and key heads against the formula in 64 bits, and with the cache write in the same launch
against the two calls, byte for byte."""

from __future__ import annotations

import numpy as np
import pytest

import _attention as A

pytestmark = pytest.mark.gpu


def _ints(cuda, values):
    import torch

    return torch.tensor(values, dtype=torch.int32, device=cuda)


def _prefix(counts):
    return [0, *np.cumsum(counts).tolist()]


def turned(x, position, frequencies, norm, eps, interleaved):
    """(result, bound of its fp32 computation) of rows x [rows, heads, dim] in 64 bits.

    Bound: the factor of the norm is off by the roundings of a sum of eight values per lane and five levels, a square
    root, a quotient and two products, 32 2^-24 at most; cosines and sines by the angle's rounding to 2^-26 of a turn,
    which is 2^-23.3, and 2^-22.4 of their own: 2^-21 at most; both apply to the two values of a pair."""
    x = np.asarray(x, dtype=np.float64)
    if norm is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(norm, dtype=np.float64)
    half = len(frequencies)
    angle = np.asarray(position, dtype=np.float64)[:, None, None] * np.asarray(frequencies, dtype=np.float64)
    cos, sin = np.cos(angle), np.sin(angle)
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (
        slice(0, half), slice(half, 2 * half))
    a, b = x[..., first], x[..., second]
    out, size = x.copy(), np.abs(x)
    out[..., first], out[..., second] = a * cos - b * sin, b * cos + a * sin
    size[..., first] = size[..., second] = np.abs(a) + np.abs(b)
    return out, size * (2.0 ** -21 + 32 * 2.0 ** -24)


def check(actual, expected, bound, dtype, what=""):
    actual = actual.double().cpu().numpy()
    # a result's rounding to its type; below the type's normal numbers half their distance, 2^-25 at most
    limit = bound * (1 + A.UNIT[dtype]) + A.UNIT[dtype] * np.abs(expected) + (2.0 ** -25 if dtype == "float16" else 1e-38)
    bad = ~(np.abs(actual - expected) <= limit)
    if bad.any():
        at = tuple(np.argwhere(bad)[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.size} off; first at {at}: {actual[at]!r} vs "
                             f"{expected[at]!r}, limit {limit[at]:.3g}")


def _positions(past, counts):
    return np.concatenate([p + np.arange(c) for p, c in zip(past, counts)])


CASES = [(64, 64, 3, 3, False), (64, 16, 4, 2, True), (128, 128, 6, 2, False), (128, 64, 1, 1, False),
         (256, 256, 5, 1, True), (256, 32, 2, 2, False), (128, 128, 17, 1, True)]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("dim,rotary,heads,kv,interleaved", CASES)
def test_against_the_formula(cuda, dtype, dim, rotary, heads, kv, interleaved):
    """Ragged rows, a sequence without any, far positions, padding behind the last sequence; with and without norms."""
    import torch
    from ivonar_amd import attention

    counts, past = [1, 0, 37, 5], [0, 3, 130000, 2 ** 20]
    rows, padding = sum(counts), 3
    generator = torch.Generator().manual_seed(dim + rotary)
    q = (torch.randn(rows + padding, heads, dim, generator=generator) * 3).to(getattr(torch, dtype)).to(cuda)
    k = torch.randn(rows + padding, kv, dim, generator=generator).to(getattr(torch, dtype)).to(cuda)
    weights = [1 + 0.3 * torch.randn(dim, generator=generator) for _ in range(2)]
    frequencies = attention.rotary_frequencies(rotary, 10000.0, device=cuda)
    offsets = _ints(cuda, _prefix(counts))
    for norms in ((None, None), tuple(weights), (weights[0], None)):
        on_device = [None if w is None else w.to(cuda) for w in norms]
        got = attention.rotate(q, k, _ints(cuda, past), frequencies, offsets, *on_device, eps=1e-5,
                               interleaved=interleaved)
        for x, y, weight in zip((q, k), got, norms):
            assert y.dtype is x.dtype and y.shape == x.shape
            assert not y[rows:].any()
            expected = turned(x[:rows].double().cpu().numpy(), _positions(past, counts), frequencies.cpu().numpy(),
                              None if weight is None else weight.numpy(), 1e-5, interleaved)
            check(y[:rows], *expected, dtype)


def test_one_row_each_and_position_zero(cuda):
    """Without offsets every sequence has a row; at position zero nothing turns, value for value."""
    import torch
    from ivonar_amd import attention

    q, k = torch.randn(200, 4, 128, device=cuda), torch.randn(200, 2, 128, device=cuda)
    frequencies = attention.rotary_frequencies(128, 500000.0, device=cuda)
    past = torch.arange(200, dtype=torch.int32, device=cuda) * 7
    got = attention.rotate(q, k, past, frequencies)
    for x, y in zip((q, k), got):
        expected = turned(x.double().cpu().numpy(), past.cpu().numpy(), frequencies.cpu().numpy(), None, 0, False)
        check(y, *expected, "float32")
    got = attention.rotate(q, k, torch.zeros_like(past), frequencies)
    assert torch.equal(got[0], q) and torch.equal(got[1], k)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_in_place_and_strided(cuda, dtype, interleaved):
    """Parts of one projection's output, off every alignment, read in place and replaced; what lies beside them stays."""
    import torch
    from ivonar_amd import attention

    heads, kv, dim, rows = 5, 2, 64, 33
    frequencies = attention.rotary_frequencies(32, device=cuda)
    weight = torch.rand(dim, device=cuda) + 0.5
    past = _ints(cuda, [11])
    offsets = _ints(cuda, [0, rows])
    for offset in (0, 1, 4, 8):
        fused = torch.randn(rows, (heads + 2 * kv) * dim + 24, device=cuda).to(getattr(torch, dtype))
        before = fused.clone()
        q = fused[:, offset:offset + heads * dim].unflatten(1, (heads, dim))
        k = fused[:, offset + heads * dim:offset + (heads + kv) * dim].unflatten(1, (kv, dim))
        expected = attention.rotate(q.clone(), k.clone(), past, frequencies, offsets, weight, weight,
                                    interleaved=interleaved)
        fresh = attention.rotate(q, k, past, frequencies, offsets, weight, weight, interleaved=interleaved)
        got = attention.rotate(q, k, past, frequencies, offsets, weight, weight, interleaved=interleaved, out=(q, k))
        assert got[0] is q and got[1] is k
        for x, y, z in zip(expected, fresh, got):
            assert torch.equal(x, y) and torch.equal(x, z), offset
        assert torch.equal(fused[:, offset + (heads + kv) * dim:], before[:, offset + (heads + kv) * dim:])
        assert torch.equal(fused[:, :offset], before[:, :offset])
    # heads apart from tokens
    q, k = (torch.randn(n, rows, dim, device=cuda).transpose(0, 1) for n in (heads, kv))
    got = attention.rotate(q, k, past, frequencies, offsets, interleaved=interleaved)
    expected = attention.rotate(q.contiguous(), k.contiguous(), past, frequencies, offsets, interleaved=interleaved)
    assert torch.equal(got[0], expected[0]) and torch.equal(got[1], expected[1])


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("dim,heads,kv,page", [(64, 6, 3, 32), (128, 8, 2, 64), (256, 1, 1, 128), (128, 40, 40, 32)])
def test_write_equals_the_two_calls(cuda, rng, dtype, dim, heads, kv, page):
    """Ragged rows over tiles and pages, entries without a page, a negative past, padding: q and every byte of the
    cache are those of rotate and cache_write."""
    import torch
    from ivonar_amd import attention

    counts, past = [1, 0, 77, 33, 2], [5, 9, 0, 31, -4]
    total, table = A.place([max(1, p + c) for p, c in zip(past, counts)], page, rng)
    table[2, 1] = -1
    rows = sum(counts) + 2
    kind = getattr(torch, dtype)
    q, k, v = (torch.randn(rows, n, dim, device=cuda).to(kind) for n in (heads, kv, kv))
    k[3, 0, 5] = float("nan")
    v[4, 0, 1] = float("inf")
    weight = torch.rand(dim, device=cuda) + 0.5
    frequencies = attention.rotary_frequencies(dim, device=cuda)
    at = torch.from_numpy(table).to(cuda), _ints(cuda, past)
    offsets = _ints(cuda, _prefix(counts))
    for interleaved in (False, True):
        pages = attention.cache_pages(total, kv, dim, page, cuda)
        pages.copy_(torch.randint(0, 256, pages.shape, dtype=torch.uint8))
        expected_pages = pages.clone()
        q_expected, k_turned = attention.rotate(q, k, at[1], frequencies, offsets, weight, weight,
                                                interleaved=interleaved)
        attention.cache_write(expected_pages, k_turned, v, *at, offsets)
        got = attention.rotate_write(pages, q, k, v, *at, frequencies, offsets, weight, weight, interleaved=interleaved)
        assert torch.equal(got, q_expected)
        assert torch.equal(pages, expected_pages)


def test_not_numbers_stay_in_their_pairs(cuda):
    """Without a norm an infinity or NaN reaches the other half of its pair and nothing else; dims that are not rotated
    keep theirs."""
    import torch
    from ivonar_amd import attention

    q = torch.ones(1, 2, 64, device=cuda)
    q[0, 0, 3], q[0, 0, 40], q[0, 1, 50] = float("inf"), float("nan"), -float("inf")
    got = attention.rotate(q, torch.ones(1, 1, 64, device=cuda), _ints(cuda, [5]),
                           attention.rotary_frequencies(32, device=cuda))[0]
    odd = ~torch.isfinite(got)
    assert odd[0, 0].nonzero().flatten().tolist() == [3, 19, 40] and odd[0, 1].nonzero().flatten().tolist() == [50]
    assert got[0, 1, 50] == -float("inf")


@pytest.mark.parametrize("rows", [1, 4096, 70000])
def test_many_rows(cuda, rows):
    """Blocks that take one head each, and blocks that take all of a token's; rows at the ends and between."""
    import torch
    from ivonar_amd import attention

    q, k = torch.randn(rows, 7, 64, device=cuda).half(), torch.randn(rows, 7, 64, device=cuda).half()
    frequencies = attention.rotary_frequencies(64, device=cuda)
    got = attention.rotate(q, k, _ints(cuda, [40]), frequencies, _ints(cuda, [0, rows]))
    some = sorted({0, rows // 2, rows - 1, *range(0, rows, max(1, rows // 50))})
    for x, y in zip((q, k), got):
        expected = turned(x[some].double().cpu().numpy(), 40 + np.array(some), frequencies.cpu().numpy(), None, 0, False)
        check(y[some], *expected, "float16")


def test_captured(cuda):
    """Replays with other values and positions in place, with eager work between them."""
    import torch
    from ivonar_amd import attention

    q, k, v = (torch.randn(8, n, 128, device=cuda).bfloat16() for n in (4, 2, 2))
    pages = attention.cache_pages(8, 2, 128, 32, cuda)
    table = torch.arange(8, dtype=torch.int32, device=cuda).view(8, 1)
    past = torch.zeros(8, dtype=torch.int32, device=cuda)
    frequencies = attention.rotary_frequencies(128, device=cuda)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        turned_q, turned_k = attention.rotate(q, k, past, frequencies)
        written_q = attention.rotate_write(pages, q, k, v, table, past, frequencies)
    for replay in range(4):
        q.copy_(torch.randn_like(q, dtype=torch.float32))
        k.copy_(torch.randn_like(k, dtype=torch.float32))
        past.fill_(3 * replay)
        torch.cuda.synchronize()
        graph.replay()
        expected = attention.rotate(q, k, past, frequencies)
        other = torch.zeros_like(pages)
        attention.cache_write(other, expected[1], v, table, past)
        assert torch.equal(turned_q, expected[0]) and torch.equal(turned_k, expected[1])
        assert torch.equal(written_q, expected[0])
        got, kept = (attention.cache_read(p, table, past, None, 8) for p in (pages, other))
        assert torch.equal(got[0], kept[0]) and torch.equal(got[1], kept[1])


def test_refusals(cuda):
    import torch
    from ivonar_amd import attention
    from ivonar_amd.runtime import KernelError

    q, k = torch.zeros(4, 4, 64, device=cuda), torch.zeros(4, 2, 64, device=cuda)
    past, frequencies, offsets = _ints(cuda, [0]), attention.rotary_frequencies(64, device=cuda), _ints(cuda, [0, 4])
    weight = torch.ones(64, device=cuda)
    pages, table = attention.cache_pages(1, 2, 64, 32, cuda), _ints(cuda, [[0]])
    good = dict(q=q, k=k, past=past, frequencies=frequencies, offsets=offsets, q_norm=weight, k_norm=weight)
    attention.rotate(**good)
    attention.rotate_write(pages, v=k, table=table, **good)
    bad = (("q", q[:3]), ("q", q[..., :32]), ("q", q.half()), ("q", q.double()), ("q", q[:, :0]), ("q", q.cpu()),
           ("k", k.flatten(1)), ("k", k[:, :0]), ("past", past.long()), ("past", past[0]), ("past", _ints(cuda, [0, 0])),
           ("offsets", None), ("offsets", offsets.long()), ("frequencies", frequencies.double()),
           ("frequencies", frequencies[:4]), ("frequencies", frequencies.repeat(2)), ("frequencies", frequencies[::2]),
           ("frequencies", frequencies[:0]), ("q_norm", weight.half()), ("k_norm", weight[:32]), ("eps", -1.0),
           ("eps", float("nan")))
    for name, value in bad:
        with pytest.raises(KernelError):
            attention.rotate(**{**good, name: value})
        with pytest.raises(KernelError):
            attention.rotate_write(pages, v=k, table=table, **{**good, name: value})
    for out in ((q[:3], k), (q, k.half()), (q.transpose(1, 2).contiguous().transpose(1, 2), k)):
        with pytest.raises(KernelError):
            attention.rotate(**good, out=out)
    for name, value in (("v", k[:3]), ("v", k.half()), ("table", table.long()), ("pages", pages[..., :-2]),
                        ("pages", pages.float()), ("table", _ints(cuda, [[0], [0]])), ("out", q[:, :2])):
        with pytest.raises(KernelError):
            attention.rotate_write(**{**good, "pages": pages, "v": k, "table": table, name: value})
    for values in ((24, 1e4, 1.0), (0, 1e4, 1.0), (64, 0.0, 1.0), (64, 1e4, 0.0), (64, float("inf"), 1.0)):
        with pytest.raises(KernelError):
            attention.rotary_frequencies(*values, device=cuda)
    empty = attention.rotate(q[:0], k[:0], past, frequencies, _ints(cuda, [0, 0]))
    assert empty[0].shape == (0, 4, 64) and empty[1].shape == (0, 2, 64)
