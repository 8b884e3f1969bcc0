"""Attention within packed prompts against a plain 64-bit implementation."""

from __future__ import annotations

import numpy as np
import pytest

import _attention as A

pytestmark = pytest.mark.gpu

# One term of the type for a weight: half a unit in its last place.
WEIGHT = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def _ints(cuda, values):
    import torch

    return torch.tensor(values, dtype=torch.int32, device=cuda)


def _inputs(cuda, rng, rows, heads, kv_heads, dim, dtype):
    import torch

    return [torch.from_numpy(rng.standard_normal((rows, h, dim)).astype(np.float32)).to(cuda).to(getattr(torch, dtype))
            for h in (heads, kv_heads, kv_heads)]


def _check(out, q, k, v, counts, dtype, **options):
    """Every sequence against its own rows; weights below 2^-24 of fp16 (times the largest, which may be 2^8 higher)
    lose up to 2^-25 of it, less than the bound's other terms leave for each key."""
    q, k, v, got = (x.float().cpu().numpy() for x in (q, k, v, out))
    start = 0
    for b, count in enumerate(counts):
        part = slice(start, start + count)
        start += count
        result = A.attend(q[part], k[part], v[part], 0, **options)
        A.check(got[part], *result, dtype, count, q.shape[-1], f"sequence {b}", weight_unit=WEIGHT[dtype])


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 2, 2), (64, 6, 2), (128, 3, 1), (128, 8, 8), (256, 2, 1)])
def test_ragged(cuda, rng, dtype, dim, heads, kv_heads):
    """Lengths of zero and one, and around the ends of the row and key tiles."""
    from ivonar_amd import attention

    counts = [1, 0, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200]
    q, k, v = _inputs(cuda, rng, sum(counts), heads, kv_heads, dim, dtype)
    out = attention.window_attention(q, k, v, _ints(cuda, [0, *np.cumsum(counts).tolist()]))
    _check(out, q, k, v, counts, dtype)


@pytest.mark.parametrize("rows", [1, 36, 300, 513])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_one_sequence(cuda, rng, rows, dim):
    from ivonar_amd import attention

    q, k, v = _inputs(cuda, rng, rows, 4, 2, dim, "bfloat16")
    _check(attention.window_attention(q, k, v), q, k, v, [rows], "bfloat16")
    _check(attention.window_attention(q, k, v, scale=0.7), q, k, v, [rows], "bfloat16", scale=0.7)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (5, 1), (64, 4), (65, 70), (200, 129), (1000, 4), (7, 600),
                                          (64, 0), (1 << 30, 1 << 30)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_window_and_sinks(cuda, rng, window, sinks, dim):
    from ivonar_amd import attention

    counts = [450, 64, 3]
    q, k, v = _inputs(cuda, rng, sum(counts), 2, 1, dim, "float16")
    out = attention.window_attention(q, k, v, _ints(cuda, [0, *np.cumsum(counts).tolist()]), window, sinks)
    _check(out, q, k, v, counts, "float16", window=window, sinks=sinks)


def test_rows_of_no_sequence(cuda, rng):
    import torch
    from ivonar_amd import attention

    q, k, v = _inputs(cuda, rng, 300, 3, 1, 64, "bfloat16")
    out = torch.full_like(q, float("nan"))
    attention.window_attention(q, k, v, _ints(cuda, [5, 150, 150, 290]), out=out)
    assert not out[:5].any() and not out[290:].any()
    _check(out[5:290], q[5:290], k[5:290], v[5:290], [145, 0, 140], "bfloat16")
    assert not attention.window_attention(q, k, v, _ints(cuda, [0])).any()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_strided(cuda, rng, dtype):
    """q, k and v as parts of one projection's output, aligned or not, and heads apart from tokens."""
    import torch
    from ivonar_amd import attention

    for offset in (0, 8, 1, 4):
        fused = torch.randn(150, 8 * 64 + 8, device=cuda).to(getattr(torch, dtype))
        q, k, v = (fused[:, offset + a:offset + b].unflatten(1, (-1, 64)) for a, b in ((0, 256), (256, 384), (384, 512)))
        expected = attention.window_attention(q.contiguous(), k.contiguous(), v.contiguous())
        assert torch.equal(attention.window_attention(q, k, v), expected)
        _check(expected, q, k, v, [150], dtype)
    q, k, v = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in _inputs(cuda, rng, 150, 4, 2, 128, dtype))
    _check(attention.window_attention(q, k, v), q, k, v, [150], dtype)
    one = k[:1].expand(150, 2, 128)  # every row the same: stride 0
    _check(attention.window_attention(q, one, one), q, one, one, [150], dtype)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_values_that_are_no_finite_numbers(cuda, rng, dtype, dim):
    """They reach the rows that see them, in their dims, as in the formula, and no others; not even the padding of
    another sequence."""
    import torch
    from ivonar_amd import attention

    q, k, v = _inputs(cuda, rng, 340, 2, 1, dim, dtype)
    k[:, :, 0] = 0
    bad = {70: np.inf, 133: -np.inf, 140: np.nan, 339: np.nan}
    for row, value in bad.items():
        v[row, 0, 3] = value
    k[200, 0, 0] = np.inf  # of q: a logit of +-infinity, whose row is no number where it sees it
    k[339, 0, 0] = np.nan
    offsets = _ints(cuda, [0, 250, 339, 340])
    for window, sinks in ((0, 0), (40, 2)):
        out = attention.window_attention(q, k, v, offsets, window, sinks).float().cpu().numpy()
        clean_v, clean_k = v.clone(), k.clone()
        for row in bad:
            clean_v[row, 0, 3] = 0
        clean_k[200, 0, 0] = clean_k[339, 0, 0] = 0
        clean = attention.window_attention(q, clean_k, clean_v, offsets, window, sinks).float().cpu().numpy()
        for i in range(250):
            seen = A.visible(i, 250, window, sinks)
            if seen[200]:
                # an infinite logit: +inf - inf is no number; -inf alone takes its weight away
                for h in range(2):
                    if float(q[i, h, 0]) > 0:
                        assert np.isnan(out[i, h]).all(), i
                continue
            rest = np.arange(dim) != 3
            assert np.array_equal(out[i][:, rest], clean[i][:, rest]), i
            values = [bad[row] for row in bad if row < 250 and seen[row]]
            if not values:
                assert np.array_equal(out[i], clean[i]), i
            elif len(set(map(str, values))) > 1 or np.isnan(values[0]):
                assert np.isnan(out[i][:, 3]).all(), i
            else:
                assert (out[i][:, 3] == values[0]).all(), i
        assert np.array_equal(out[250:339], clean[250:339])
        assert np.isnan(out[339]).all()


def test_large_logits(cuda, rng):
    from ivonar_amd import attention

    q, k, v = _inputs(cuda, rng, 400, 2, 1, 64, "bfloat16")
    k *= 16
    q[..., 5] *= 64
    _check(attention.window_attention(q, k, v), q, k, v, [400], "bfloat16")
    _check(attention.window_attention(q, k, v, window=100, sinks=3), q, k, v, [400], "bfloat16", window=100, sinks=3)


def test_long_prompt(cuda, rng):
    """A few rows of a long prompt, with and without a window."""
    import torch
    from ivonar_amd import attention

    q, k, v = _inputs(cuda, rng, 5000, 2, 1, 128, "float16")
    rows = [0, 127, 128, 2047, 3333, 4999]
    for window, sinks in ((0, 0), (700, 5)):
        out = attention.window_attention(q, k, v, None, window, sinks).float().cpu().numpy()
        kept = [x.float().cpu().numpy() for x in (q, k, v)]
        for row in rows:
            result = A.attend(kept[0][row:row + 1], kept[1][:row + 1], kept[2][:row + 1], row, window, sinks)
            A.check(out[row:row + 1], *result, "float16", row + 1, 128, f"row {row}", weight_unit=WEIGHT["float16"])


def test_in_a_graph(cuda, rng):
    import torch
    from ivonar_amd import attention

    q, k, v = _inputs(cuda, rng, 500, 4, 2, 64, "bfloat16")
    offsets, out = _ints(cuda, [0, 100, 500]), torch.empty_like(q)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        attention.window_attention(q, k, v, offsets, 64, 4, out=out)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        attention.window_attention(q, k, v, offsets, 64, 4, out=out)
    for turn in range(4):
        offsets[1] = 100 + 50 * turn
        k.normal_()
        graph.replay()
        replayed = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(attention.window_attention(q, k, v, offsets, 64, 4), replayed)


def test_refusals(cuda, rng):
    import torch
    from ivonar_amd import attention
    from ivonar_amd.runtime import KernelError, library

    q, k, v = _inputs(cuda, rng, 10, 4, 2, 64, "float16")
    good = dict(q=q, k=k, v=v)
    attention.window_attention(**good)
    for name, value in (("q", q.float()), ("q", q.bfloat16()), ("q", q[:9]), ("q", q[:, :3]), ("q", q[..., :32]),
                        ("q", q.cpu()), ("k", k[:, :1]), ("k", k[0]), ("v", v.bfloat16()), ("v", v[:9]),
                        ("k", k.repeat(1, 1, 2)[..., ::2]), ("window", -1), ("sinks", -2), ("scale", 0.0),
                        ("scale", float("inf")), ("offsets", torch.zeros(0, dtype=torch.int32, device=cuda)),
                        ("offsets", torch.zeros(2, device=cuda)), ("offsets", _ints("cpu", [0, 10])), ("out", q[:, :2]),
                        ("out", q.bfloat16())):
        with pytest.raises(KernelError):
            attention.window_attention(**{**good, name: value})
    with pytest.raises(KernelError):
        attention.window_attention(q.float(), k.float(), v.float())
    assert attention.window_attention(q[:0], k[:0], v[:0]).shape == (0, 4, 64)
    lib = library()

    def call(address=0, dtype=1, strides=(256, 64, 128, 64, 128, 64), heads=4, sequences=1, scale=0.1):
        return lib.ivonar_window_attention(0, q.data_ptr() + address, k.data_ptr(), v.data_ptr(), dtype, *strides, heads,
                                           2, 64, 10, None, sequences, 0, 0, scale, torch.empty_like(q).data_ptr())

    assert call() == 0
    for bad in (dict(address=2), dict(dtype=0), dict(dtype=3), dict(strides=(257, 64, 128, 64, 128, 64)),
                dict(strides=(256, 64, 1 << 23, 64, 128, 64)), dict(strides=(256, 64, 128, 64, -128, 64)),
                dict(heads=3), dict(sequences=2), dict(scale=0.0)):
        assert call(**bad) != 0


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("spread", [1.0, 3.0, 40.0])
def test_infinities_at_any_key(cuda, rng, dtype, dim, spread):
    """An infinite value that a row sees makes its sum infinite, in whichever of the row's tiles the key lies and
    however small its weight is; every other number is what it is without them."""
    from ivonar_amd import attention

    q, k, v = _inputs(cuda, rng, 340, 2, 1, dim, dtype)
    q *= spread  # how far the weights are apart
    bad = [(0, 1, np.inf), (2, 2, -np.inf), (3, 3, np.inf), (70, dim - 1, -np.inf), (200, 40, np.inf),
           (290, 1, np.inf), (300, 2, np.inf), (310, 9, np.nan)]
    clean_v = v.clone()
    for row, column, value in bad:
        v[row, 0, column] = value
        clean_v[row, 0, column] = 0
    for window, sinks in ((0, 0), (40, 0), (100, 2)):
        expected = attention.window_attention(q, k, clean_v, None, window, sinks).float().cpu().numpy()
        for i in range(340):
            seen = A.visible(i, 340, window, sinks)
            for row, column, value in bad:
                if seen[row]:
                    with np.errstate(invalid="ignore"):  # of both signs: no number
                        expected[i, :, column] += value
        out = attention.window_attention(q, k, v, None, window, sinks).float().cpu().numpy()
        np.testing.assert_array_equal(out, expected, err_msg=f"window {window}, sinks {sinks}")


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_logits_past_the_integers(cuda, rng, dtype, dim):
    """Logits so large that fp32 holds them in steps of far more than one: the largest takes all the weight, and rows
    next to such a row come out as they do without it."""
    import torch
    from ivonar_amd import attention

    q, k, v = _inputs(cuda, rng, 200, 2, 1, dim, dtype)
    order = rng.permutation(200)
    k[:, 0, 0] = torch.from_numpy(order.astype(np.float32)).to(k)
    large = q.clone()
    large[1::3] = 0
    large[1::3, 0, 0], large[1::3, 1, 0] = 2.0 ** 15, -2.0 ** 15
    for window, sinks in ((0, 0), (50, 4)):
        for scale in (2.0 ** 10, 2.0 ** 16, 2.0 ** 30):  # logits from 2^25 to 2^52
            out = attention.window_attention(large, k, v, None, window, sinks, scale)
            for i in range(1, 200, 3):
                keys = np.flatnonzero(A.visible(i, 200, window, sinks))
                for head, best in enumerate((keys[order[keys].argmax()], keys[order[keys].argmin()])):
                    assert torch.equal(out[i, head], v[best, 0]), (scale, i, head)
        # the other rows' logits are common ones: as if there were no large ones
        small = q * 2.0 ** -10
        small[1::3] = large[1::3]
        others = np.flatnonzero(np.arange(200) % 3 != 1)
        out = attention.window_attention(small, k, v, None, window, sinks, 2.0 ** 10)
        small[1::3] = 0
        assert torch.equal(out[others], attention.window_attention(small, k, v, None, window, sinks, 2.0 ** 10)[others])


def test_misaligned_output_is_named(cuda, rng):
    import torch
    from ivonar_amd import attention
    from ivonar_amd.runtime import KernelError

    q, k, v = _inputs(cuda, rng, 10, 4, 2, 64, "float16")
    out = torch.empty(10 * 4 * 64 + 4, dtype=torch.float16, device=cuda)[4:].view(10, 4, 64)
    with pytest.raises(KernelError, match="out .*16 bytes"):
        attention.window_attention(q, k, v, out=out)


def test_results_past_2_to_31_elements(cuda):
    import torch
    from ivonar_amd import attention

    rows, heads, dim = 131200, 64, 256
    q = torch.zeros(rows, heads, dim, dtype=torch.bfloat16, device=cuda)
    v = torch.randn(rows, 1, dim, device=cuda).bfloat16()
    out = attention.window_attention(q, v, v, window=1)  # every row sees itself
    for start in range(0, rows, 8200):
        part = slice(start, start + 8200)
        assert torch.equal(out[part], v[part].expand(8200, heads, dim))
