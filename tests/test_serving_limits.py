"""Limits of the serving calls that are checked, or planned for, without a device."""

from __future__ import annotations

import torch

from ivonar_amd.runtime import library

INVALID = 1  # hipErrorInvalidValue
P = 4096     # an address that no refused call looks at


def test_temperatures_whose_inverse_is_out_of_range():
    """Half-way differences are multiplied by 2 log2(e) / T, which has to be a number."""
    def call(temperature):
        return library().ivonar_log_probabilities(None, P, 0, 100, 1, 100, P, 5, temperature, P, P, P, P, None, 0)

    for temperature in (5.9e-39, 8e-39, 1.1e-38):
        assert call(temperature) == INVALID
    if not torch.cuda.is_available():
        assert call(1.2e-38) != INVALID  # past the checks, and finds no device


def test_tails_are_shared_out_where_no_prefix_is_known():
    """A split tail needs room for its parts, beside the prefix's; a tail of a few tiles needs none."""
    work = library().ivonar_prefix_attention_work
    sizes = (2, 32, 8, 128, None, 8, 8, 1)  # eight rows, one group
    whole, part = 8 * 8 * (128 + 2) * 4, 16  # of a row tile of each head; the groups' shared tokens
    for longest in (2000, 20000, 130000):
        assert work(*sizes, longest - 21, longest) < work(*sizes, -1, longest)
        prefix = work(*sizes, longest, longest)  # tails of nothing
        tails = work(*sizes, 0, longest) - work(*sizes, 0, 0)  # of all keys
        assert tails > 0 and tails % (8 * whole) == 0
        assert work(*sizes, -1, longest) == prefix + tails
        assert (prefix - part) % whole == 0


def test_fork_writes_into_none_of_its_inputs():
    good = [P, P, 40, 64, P, 4, P, 2, 2 * P, 3, 3 * P, 4 * P, P, P]
    for at, value in ((10, P), (11, P), (11, 2 * P)):  # the table, the lengths, the parents
        args = list(good)
        args[at] = value
        assert library().ivonar_page_fork(None, *args) == INVALID
    if not torch.cuda.is_available():
        assert library().ivonar_page_fork(None, *good) != INVALID
