"""prefix_attention as it is called without hints: long keys of a sequence's own, in and outside groups."""

from __future__ import annotations

import pytest

from test_gpu_prefix_attention import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,heads,kv,dim", [("float32", 4, 4, 64), ("bfloat16", 8, 2, 128), ("float16", 4, 1, 256)])
@pytest.mark.parametrize("rows", [1, 3])
def test_long_tails_without_hints(cuda, rng, dtype, heads, kv, dim, rows, monkeypatch):
    """Tails of up to 126 tiles, at most 16 parts beside the prefix's, shared out between blocks by default too."""
    from ivonar_amd import attention

    sequences = [(None, 0, 4010, rows), (0, 3, 3900, rows), (0, 3, rows, rows), (0, 3, 2001, rows), (None, 0, rows, rows)]
    batch = Batch(cuda, rng, sequences, heads, kv, dim, 32, dtype)
    batch.groups = [1, 4]
    needs, work = [], attention._prefix_workspace

    def recorded(*sizes):
        needs.append(work(*sizes))
        return needs[-1]

    monkeypatch.setattr(attention, "_prefix_workspace", recorded)
    for hints in ({}, {"max_length": 4010}, {"max_prefix": 96}, {"max_prefix": 1 << 20}):
        batch.check(batch.run(**hints), str(hints))
    assert needs[0] > needs[3] and needs[1] > needs[3]  # room for the tails' parts
