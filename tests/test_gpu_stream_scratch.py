"""The first calls on a new stream, whose counters are cleared before them."""

from __future__ import annotations

import ctypes
import os

import pytest

pytestmark = pytest.mark.gpu


def test_first_calls_on_a_new_stream(cuda):
    """With work under way on the null stream, where a clear that nobody waits for would end among the calls."""
    import torch
    from ivonar_amd import attention

    runtime = ctypes.CDLL(os.path.join(os.path.dirname(torch.__file__), "lib", "libamdhip64.so"))
    generator = torch.Generator().manual_seed(1)
    pages = attention.cache_pages(63, 2, 128, 64, cuda)
    table = torch.arange(63, dtype=torch.int32, device=cuda)[None]
    k, v = (torch.randn(4000, 2, 128, generator=generator).to(cuda) for _ in range(2))
    ints = [torch.tensor(values, dtype=torch.int32, device=cuda) for values in ([0], [0, 4000], [4000])]
    attention.cache_write(pages, k, v, table, ints[0], ints[1])
    q = torch.randn(1, 8, 128, generator=generator).to(cuda)
    expected = attention.cache_attention(q, pages, table, ints[2])
    square = torch.randn(4096, 4096, device=cuda)
    for _ in range(2):
        handle = ctypes.c_void_p()
        assert runtime.hipStreamCreateWithFlags(ctypes.byref(handle), 1) == 0  # one that does not wait for the null stream
        stream = torch.cuda.ExternalStream(handle.value)
        out = torch.zeros(200, 1, 8, 128, device=cuda)
        torch.cuda.synchronize()
        for _ in range(8):
            square @ square
        with torch.cuda.stream(stream):
            for one in out:
                attention.cache_attention(q, pages, table, ints[2], out=one)
        torch.cuda.synchronize()
        assert (out == expected).all()
