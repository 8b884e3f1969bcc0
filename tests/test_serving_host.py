"""What the calls for rotations, pages, shared prefixes and scores check without a device, and the tests' own plain pool."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import _paging
from ivonar_amd import attention, paging, sampling
from ivonar_amd.runtime import KernelError, SIGNATURES, library

INVALID = 1  # hipErrorInvalidValue, from the entry's own checks: a launch would fail otherwise here
P = 4096     # an address that no refused call looks at


def _refused(name, good, changes):
    """Every change of one argument is refused; `good` itself gets past the checks (and finds no device)."""
    function = getattr(library(), name)
    for at, value in changes:
        args = list(good)
        args[at] = value
        assert function(None, *args) == INVALID, (name, at, value)
    if not torch.cuda.is_available():
        assert function(None, *good) != INVALID


def test_entry_points_are_declared():
    for name in ("ivonar_rotate", "ivonar_rotate_write", "ivonar_page_reserve", "ivonar_page_release", "ivonar_page_fork",
                 "ivonar_page_compact", "ivonar_page_copy", "ivonar_prefix_attention", "ivonar_log_probabilities"):
        assert name in SIGNATURES and hasattr(library(), name)


def test_rotate_entries_refuse():
    # q, k, dtype, strides, heads, kv_heads, dim, rows, past, offsets, sequences, frequencies, rotary, .., q_out, k_out
    good = [P, P, 0, 256, 64, 128, 64, 4, 2, 64, 3, P, P, 1, P, 64, 0, None, None, 1e-6, P, P, 256, 64, 128, 64]
    _refused("ivonar_rotate", good, [(0, None), (1, None), (2, 3), (2, -1), (7, 0), (8, 0), (8, 65536), (9, 96), (10, -1),
                                     (11, None), (12, None), (13, -1), (14, None), (15, 0), (15, 24), (15, 80), (15, -16),
                                     (20, None), (21, None)])
    good = [P, P, P, 0, 256, 64, 128, 64, 128, 64, 4, 3, P, 5, 2, 2, 64, P, 4, P, P, 1, P, 64, 0, None, None, 1e-6, P, 256,
            64]
    _refused("ivonar_rotate_write", good, [(0, None), (1, None), (2, None), (3, 3), (10, 0), (12, P + 8), (12, None),
                                           (13, 0), (14, 0), (15, 3), (16, 32), (17, None), (18, 0), (18, 1 << 25),
                                           (19, None), (20, None), (22, None), (23, 40), (28, None)])


def test_page_entries_refuse():
    pool = [P, P, 40, 64]
    of_pool = [(0, None), (1, None), (2, 0), (2, (1 << 27) + 1), (3, 48), (3, 16), (3, 0), (4, None), (5, 0), (5, 1 << 25)]
    _refused("ivonar_page_reserve", [*pool, P, 4, P, P, 2, P], of_pool + [(6, None), (7, None), (8, -1), (9, None)])
    _refused("ivonar_page_release", [*pool, P, 4, None, None, 2], of_pool + [(8, -1), (8, 1 << 30)])
    _refused("ivonar_page_fork", [*pool, P, 4, P, 2, P, 3, 2 * P, 2 * P, P, P],
             of_pool + [(6, None), (7, -1), (7, 8193), (8, None), (9, -1), (9, 1 << 30), (10, None), (10, P), (11, None),
                        (11, P), (12, None), (13, None)])
    _refused("ivonar_page_compact", [*pool, P, 4, 2, P, P, P], of_pool + [(6, -1), (7, None), (8, None), (9, None)])
    _refused("ivonar_page_copy", [P, 40, 2176, P, 3], [(0, None), (0, P + 8), (1, 0), (2, 0), (2, 8), (2, 1 << 41), (3, None),
                                                       (3, P + 4), (4, -1)])


def test_prefix_attention_entry_refuses():
    lib = library()
    sizes = (0, 4, 2, 64, None, 5, 5, 2, 100, 200)
    need = lib.ivonar_prefix_attention_work(*sizes)
    assert need > 0
    for at, value in ((0, 3), (1, 3), (1, 0), (2, 0), (3, 96), (5, -1), (6, -1), (7, -1), (7, 6)):
        assert lib.ivonar_prefix_attention_work(*sizes[:at], value, *sizes[at + 1:]) == -1
    good = [P, 0, 256, 64, 4, 5, P, 9, 2, 2, 64, P, 4, P, None, 5, P, P, 2, 0.125, 100, 200, P, P, need]
    _refused("ivonar_prefix_attention", good, [(0, None), (1, 3), (4, 3), (5, 4), (6, None), (6, P + 8), (7, 0), (8, 3),
                                               (9, 3), (10, 80), (11, None), (12, 0), (13, None), (15, 6), (16, None),
                                               (17, None), (18, -1), (18, 6), (19, 0.0), (22, None), (22, P + 8),
                                               (23, None), (23, P + 8), (24, need - 1)])


def test_score_entry_refuses():
    lib = library()
    assert lib.ivonar_log_probabilities_work(0, 1000000, 1000, 20) == 0
    assert lib.ivonar_log_probabilities_work(0, 1, 32000, 20) == 0  # one block a row
    need = lib.ivonar_log_probabilities_work(0, 1, 1000000, 20)
    assert need > 0
    for sizes in ((3, 1, 100, 5), (0, -1, 100, 5), (0, 1, 0, 0), (0, 1, 100, 65), (0, 1, 10, 11), (0, 1, 100, -1),
                  (0, 1, (1 << 30) + 1, 5)):
        assert lib.ivonar_log_probabilities_work(*sizes) == -1
    good = [P, 0, 1000000, 1, 1000000, P, 20, 1.0, P, P, P, P, P, need]
    _refused("ivonar_log_probabilities", good, [(0, None), (0, P + 2), (1, 3), (3, -1), (4, 0), (5, None), (6, 65), (6, -1),
                                                (7, 0.0), (7, -1.0), (7, float("nan")), (7, float("inf")), (7, 1e-42),
                                                (8, None), (9, None), (10, None), (11, None), (12, None), (12, P + 8),
                                                (13, need - 1)])


def test_tensors_must_be_on_a_device():
    x, ints = torch.zeros(1, 1, 64), torch.zeros(1, dtype=torch.int32)
    pages, table = attention.cache_pages(1, 1, 64, 64, "cpu"), torch.zeros(1, 1, dtype=torch.int32)
    frequencies = attention.rotary_frequencies(64, device="cpu")
    pool = paging.page_pool(4, 64, "cpu")
    for call in (lambda: attention.rotate(x, x, ints, frequencies),
                 lambda: attention.rotate_write(pages, x, x, x, table, ints, frequencies),
                 lambda: attention.prefix_attention(x, pages, table, ints, torch.zeros(2, dtype=torch.int32), ints),
                 lambda: paging.reserve(pool, table, ints, ints), lambda: paging.release(pool, table),
                 lambda: paging.fork(pool, table, ints, ints), lambda: paging.compact(pool, table),
                 lambda: paging.copy(pages, torch.zeros(1, 2, dtype=torch.int32)),
                 lambda: sampling.log_probabilities(torch.zeros(1, 8), torch.zeros(1, dtype=torch.int64))):
        with pytest.raises(KernelError):
            call()


@pytest.mark.parametrize("pages", [1, 31, 32, 33, 64, 100])
def test_a_new_pool_is_free(pages):
    pool = paging.page_pool(pages, 32, "cpu")
    assert not pool.refs.any() and pool.refs.shape == (pages,)
    assert np.array_equal(pool.free.numpy(), _paging.Pool(pages, 32).words())
    for bad in ((0, 64), (5, 33), (5, 0), (5, 16), ((1 << 27) + 1, 64)):
        with pytest.raises(KernelError):
            paging.page_pool(*bad, "cpu")


def test_frequencies():
    got = attention.rotary_frequencies(64, 10000.0, device="cpu").double()
    assert torch.allclose(got, 10000.0 ** (-torch.arange(0, 64, 2).double() / 64), rtol=2.0 ** -24)
    assert torch.allclose(attention.rotary_frequencies(64, 10000.0, 4.0, "cpu").double(), got / 4, rtol=2.0 ** -23)


def test_the_plain_pool():
    """Two children of one parent: the first takes it over, the second shares whole pages and copies the last."""
    pool, table = _paging.Pool(6, 32), np.full((1, 4), -1, dtype=np.int32)
    assert pool.reserve(table, [0], [70]) == 0 and table.tolist() == [[0, 1, 2, -1]]
    new, lengths, copies, missing = pool.fork(table, [70], [0, 0, -1])
    assert new.tolist() == [[0, 1, 2, -1], [0, 1, 3, -1], [-1] * 4] and lengths.tolist() == [70, 70, 0]
    assert copies == [(2, 3)] and missing == 0 and pool.refs.tolist() == [2, 2, 1, 1, 0, 0]
    pool.release(new, first=[0, 9, 9])
    assert pool.refs.tolist() == [1, 1, 0, 1, 0, 0]
    assert pool.compact(new) == ([(3, 2)], 3) and new[1].tolist() == [0, 1, 2, -1]
    assert pool.words().tolist() == [0b111000]
