"""What the attention module checks without a device, and the tests' own 64-bit quantiser."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import _attention as A
from ivonar_amd import attention
from ivonar_amd.runtime import KernelError, SIGNATURES, library


def test_pages_have_the_stated_size():
    for dim in attention.HEAD_DIMS:
        pages = attention.cache_pages(3, 2, dim, 128, "cpu")
        assert pages.shape == (3, 2, 4, 34 * dim) and pages.dtype == torch.uint8 and not pages.any()
    for bad in ((0, 1, 64, 64), (1, 0, 64, 64), (1, 1, 32, 64), (1, 1, 64, 96), (1, 1, 64, 8)):
        with pytest.raises(KernelError):
            attention.cache_pages(*bad, "cpu")


def test_tensors_must_be_on_a_device():
    pages = attention.cache_pages(1, 1, 64, 64, "cpu")
    table, zero = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(1, 1, 64)
    with pytest.raises(KernelError):
        attention.cache_write(pages, x, x, table, zero)
    with pytest.raises(KernelError):
        attention.cache_read(pages, table, zero, None, 1)
    with pytest.raises(KernelError):
        attention.cache_attention(x, pages, table, zero)
    with pytest.raises(KernelError):
        attention.window_attention(x.half(), x.half(), x.half())


def test_entry_points_are_declared():
    lib = library()
    for name in ("ivonar_cache_write", "ivonar_cache_read", "ivonar_cache_attention", "ivonar_window_attention"):
        assert name in SIGNATURES and hasattr(lib, name)
    # sizes that a call refuses need no workspace
    for sizes in ((3, 4, 2, 64), (0, 4, 3, 64), (0, 4, 2, 80), (0, 0, 2, 64)):
        assert lib.ivonar_cache_attention_work(*sizes, None, 1, 1, 0, 0, 100) == -1
    assert lib.ivonar_cache_attention_work(0, 4, 2, 64, None, 1, 1, -1, 0, 100) == -1
    # one block per head takes a short sequence; its result needs no workspace
    assert lib.ivonar_cache_attention_work(0, 4, 2, 64, None, 1, 1, 0, 0, 100) == 0
    assert lib.ivonar_cache_attention_work(0, 4, 2, 64, None, 1, 1, 0, 0, 100000) > 0


def test_quantiser_takes_the_nearest_value(rng):
    """Against the distances to every value of the block's grid, and the rule that places the grid."""
    x = rng.standard_normal((50, 64)) * np.exp2(rng.integers(-60, 60, (50, 1)))
    got = A.stored(x)
    blocks = x.reshape(-1, 32)
    most = np.abs(blocks).max(1)
    steps = np.exp2(A.block_exponent(most))
    assert (most / steps < 7).all() and (most / steps >= 3.5).all()
    grid = np.concatenate((A.GRID, -A.GRID)) * steps[:, None, None]
    nearest = np.abs(blocks[..., None] - grid).min(-1)
    assert np.allclose(np.abs(got.reshape(-1, 32) - blocks), nearest, rtol=1e-12, atol=0)


def test_quantiser_ties_and_odd_values():
    block = np.zeros((1, 32))
    block[0, :9] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -5]
    assert A.stored(block)[0, :9].tolist() == [6, 0, 1, 1, 2, 2, 4, 4, -4]
    block[0, 20] = np.inf
    assert np.isnan(A.stored(block)).all()
    assert not A.stored(np.zeros((1, 32))).any()
    assert A.block_exponent(np.array([0.0, 1.7499, 1.75, 6.999, 7.0, 1e300])).tolist() == [-100, -2, -1, 0, 1, 125]


@pytest.mark.parametrize("window,sinks", [(0, 0), (3, 0), (3, 2), (1, 5)])
def test_visible_keys(window, sinks):
    for position in range(-2, 9):
        expected = [j for j in range(8) if j <= position and (window == 0 or j > position - window or j < sinks)]
        assert np.flatnonzero(A.visible(position, 8, window, sinks)).tolist() == expected


@pytest.mark.parametrize("count", [1, 40])
def test_bound_notices_a_weight_of_one_term(count):
    """Weights rounded to one bfloat16 term miss the bound for two by far, and weights of two terms keep it."""
    k, v, scale = A.cancelling(300, 64)
    q = np.zeros((count, 2, 64))
    q[..., 0] = 1
    out, spread, size = A.attend(q, k, v, 300 - count, scale=scale)
    limit = A.bound(out, spread, size, "bfloat16", 300, 64, weight_unit=2.0 ** -17)

    def emulated(terms):
        got = np.zeros_like(out)
        for i in range(count):
            keys = 300 - count + i + 1
            weight = np.exp(scale * (k[:keys, 0, 0].astype(np.float64) - 1))
            rounded, rest = np.zeros(keys), weight
            for _ in range(terms):
                term = torch.from_numpy(rest).bfloat16().double().numpy()
                rounded, rest = rounded + term, rest - term
            got[i] = rounded @ v[:keys, 0] / weight.sum()
        return torch.from_numpy(got).bfloat16().double().numpy()

    assert (np.abs(emulated(1) - out) > 4 * limit).all()
    assert (np.abs(emulated(2) - out) <= limit).all()


@pytest.mark.parametrize("options", [{"page_size": 0}, {"page_size": -64}, {"window": -1}, {"window": 8, "sinks": -1},
                                     {"heads": 3}, {"capacity": 0}])
def test_decoder_refuses_what_its_calls_would(options):
    from ivonar_amd.decoder import AttentionConfig, _Attention

    with pytest.raises(KernelError):
        _Attention(AttentionConfig(**{"heads": 4, **options}), 256, 1, 32, torch.device("cpu"))
    _Attention(AttentionConfig(4, window=8, sinks=1), 256, 1, 32, torch.device("cpu"))
