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
