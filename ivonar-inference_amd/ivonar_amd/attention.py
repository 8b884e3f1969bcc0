"""Attention for a decoder of ternary layers: a key/value cache in 4 bits, and the attention that reads it.

The reference keeps fp16 keys and values and attends to them in ``attention_step`` and ``attention_tile``
(``ternary.cu:509-611``, ``:904-982``).  Here:

* ``cache_pages(pages, kv_heads, head_dim, page_size)`` -> the cache's pages, a uint8 tensor
  [pages, kv_heads, page_size / 32, 34 * head_dim];
* ``cache_write(pages, k, v, table, past, offsets)``: new tokens' keys and values, quantised as they are written;
* ``cache_read(pages, table, start, offsets, rows, dtype)`` -> (k, v): stretches of the sequences as tensors;
* ``cache_attention(q, pages, table, lengths, offsets, window, sinks)``: the last rows of each sequence (one token
  while decoding, several for a chunk of a prompt) over all of its cached tokens, or over a sliding window and the
  first few (sinks);
* ``window_attention(q, k, v, offsets, window, sinks)``: causal attention within packed prompts over their fp16 or
  bfloat16 keys and values as they are.

A cached value is a 4-bit floating-point number (0, 0.5, 1, 1.5, 2, 3, 4, 6 or a negative of them) times a power of two
that 32 neighbouring values of a head's row share: 4.25 bits per value.  A block of 32 that holds a NaN or an
infinity reads back as NaN.

``table`` [sequences, width] (int32) holds each sequence's page numbers in order; an entry outside the pages (-1, for
instance) is no page, and so is every position past the table: nothing is written there, zeros are read, and attention
does not see its tokens, so pages before a window may be handed back.  ``offsets`` (int32 [sequences + 1]) are the
rows before each sequence in a ragged batch; None stands for one row per sequence.  Rows past the last sequence's
(padding) are not written to the cache, and are zero in the results.

Index tensors stay on the device: no call reads them on the host, allocates more than its results and a workspace, or
synchronises, so all of them can be captured into a graph.  Where blocks share a sequence's keys, ``cache_attention``
counts them in the library's scratch of the stream, and under capture in that of the capture stream if it has made an
eager call before, else of the device.  So graphs captured on one stream, or an eager call on that stream and a replay
on another, must not run at the same time: their results would be undefined, and the counts they leave would spoil
later calls until the library's ``ivonar_init`` clears them.  Eager calls on different streams may overlap.
"""

from __future__ import annotations

import functools
import math

import torch
from torch import Tensor

from . import runtime
from .ops import _address
from .runtime import KernelError, check, initialise, library

TOKENS_PER_TILE = 32
HEAD_DIMS = (64, 128, 256)
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_raw_stream = torch._C._cuda_getCurrentRawStream


def cache_pages(pages: int, kv_heads: int, head_dim: int, page_size: int = 64,
                device: torch.device | str = "cuda") -> Tensor:
    """An empty cache of `pages` pages of `page_size` tokens (a power of two from 32 on) for every key/value head."""
    if head_dim not in HEAD_DIMS:
        raise KernelError(f"head_dim {head_dim} is not one of {HEAD_DIMS}")
    if page_size < TOKENS_PER_TILE or page_size & (page_size - 1):
        raise KernelError(f"page_size {page_size} is not a power of two from {TOKENS_PER_TILE} on")
    if pages <= 0 or kv_heads <= 0:
        raise KernelError("a cache needs at least one page and one head")
    return torch.zeros((pages, kv_heads, page_size // TOKENS_PER_TILE, 34 * head_dim), dtype=torch.uint8, device=device)


# The checks below read as few attributes as they can: each costs as much host time as a few instructions of the launch,
# and a decoder makes these calls once per layer and token.


def _device(first: Tensor, *others: Tensor | None) -> int:
    index = first.get_device()
    for tensor in others:
        if tensor is not None and tensor.get_device() != index:
            raise KernelError("the tensors of a call must be on one ROCm device")
    if index < 0:
        raise KernelError("attention and its cache need tensors on a ROCm device")
    if index not in runtime._initialised:
        initialise(index)
    return index


def _run(name: str, index: int, *args) -> None:
    status = getattr(library(), name)(_raw_stream(index), *args)
    if status != 0:
        check(status, name)


def _geometry(pages: Tensor, table: Tensor, what: str) -> tuple[int, int, int, int, int, int]:
    """(pages, kv_heads, tiles per page, head_dim, sequences, width) of a cache and its table."""
    shape = pages.shape
    if len(shape) != 4 or pages.dtype is not torch.uint8 or not pages.is_contiguous():
        raise KernelError(f"{what} needs pages as cache_pages() makes them")
    count, heads, tiles, size = shape
    dim = size // 34
    if dim * 34 != size or dim not in HEAD_DIMS or tiles & (tiles - 1) or not (count and heads and tiles):
        raise KernelError(f"{what} needs pages as cache_pages() makes them")
    if pages.data_ptr() & 15:
        raise KernelError(f"{what} needs pages that start on 16 bytes")
    shape = table.shape
    if len(shape) != 2 or table.dtype is not torch.int32 or not table.is_contiguous():
        raise KernelError(f"{what} needs a contiguous int32 table [sequences, width]")
    sequences, width = shape
    if width * tiles * TOKENS_PER_TILE > 1 << 30:
        raise KernelError(f"{what}: a sequence has at most 2**30 tokens")
    return count, heads, tiles, dim, sequences, width


def _index(tensor: Tensor, count: int, what: str) -> None:
    if tensor.dtype is not torch.int32 or tensor.shape != (count,) or not tensor.is_contiguous():
        raise KernelError(f"{what} must be contiguous int32 [{count}]")


def _offsets(offsets: Tensor | None, sequences: int, rows: int) -> None:
    if offsets is not None:
        _index(offsets, sequences + 1, "offsets")
    elif rows != sequences:
        raise KernelError(f"{rows} rows of {sequences} sequences need offsets")


def _rows(x: Tensor, heads: int | None, head_dim: int | None, what: str) -> tuple[int, int, int, int]:
    """(rows, heads, stride of a row, stride of a head) of x."""
    shape = x.shape
    if len(shape) != 3 or (heads is not None and shape[1] != heads) or (head_dim is not None and shape[2] != head_dim):
        raise KernelError(f"{what} must be [rows, {heads or 'heads'}, {head_dim or 'head_dim'}], not {list(shape)}")
    if x.dtype not in _DTYPES:
        raise KernelError(f"{what} must be float32, float16 or bfloat16, not {x.dtype}")
    row, head, value = x.stride()
    if value != 1:
        raise KernelError(f"{what} must have a head's values side by side")
    return shape[0], shape[1], row, head


def cache_write(pages: Tensor, k: Tensor, v: Tensor, table: Tensor, past: Tensor, offsets: Tensor | None = None) -> None:
    """Quantises rows of k and v [rows, kv_heads, head_dim] (fp32, fp16 or bfloat16, any row and head stride) into the
    cache: row r of sequence b becomes position past[b] + r - offsets[b]."""
    device = _device(pages, k, v, table, past, offsets)
    count, heads, tiles, dim, sequences, width = _geometry(pages, table, "cache_write")
    rows, _, k_row, k_head = _rows(k, heads, dim, "k")
    v_rows, _, v_row, v_head = _rows(v, heads, dim, "v")
    if v_rows != rows or v.dtype is not k.dtype:
        raise KernelError("k and v must have the same rows and type")
    _offsets(offsets, sequences, rows)
    _index(past, sequences, "past")
    if rows:
        _run("ivonar_cache_write", device, k.data_ptr(), v.data_ptr(), _DTYPES[k.dtype], k_row, k_head, v_row, v_head,
             rows, pages.data_ptr(), count, heads, tiles, dim, table.data_ptr(), width, past.data_ptr(),
             _address(offsets), sequences)


def cache_read(pages: Tensor, table: Tensor, start: Tensor | None, offsets: Tensor | None, rows: int,
               dtype: torch.dtype = torch.float32) -> tuple[Tensor, Tensor]:
    """(k, v) [rows, kv_heads, head_dim] as `dtype`: row r of sequence b is position start[b] + r - offsets[b] (start
    None: 0)."""
    device = _device(pages, table, start, offsets)
    count, heads, tiles, dim, sequences, width = _geometry(pages, table, "cache_read")
    if dtype not in _DTYPES:
        raise KernelError(f"the cache is read as float32, float16 or bfloat16, not {dtype}")
    if rows < 0:
        raise KernelError("rows must not be negative")
    _offsets(offsets, sequences, rows)
    if start is not None:
        _index(start, sequences, "start")
    k = pages.new_empty((rows, heads, dim), dtype=dtype)
    v = torch.empty_like(k)
    if rows:
        _run("ivonar_cache_read", device, pages.data_ptr(), count, heads, tiles, dim, table.data_ptr(), width,
             _address(start), _address(offsets), sequences, rows, _DTYPES[dtype], k.data_ptr(), v.data_ptr())
    return k, v


def _scale(scale: float | None, head_dim: int, window: int, sinks: int) -> float:
    if window < 0 or sinks < 0:
        raise KernelError("window and sinks must not be negative")
    if scale is None:
        return head_dim ** -0.5
    if not (scale > 0 and math.isfinite(scale)):
        raise KernelError("scale must be positive and finite")
    return float(scale)


def _output(q: Tensor, out: Tensor | None) -> Tensor:
    if out is None:
        return torch.empty_like(q, memory_format=torch.contiguous_format)
    if out.shape != q.shape or out.dtype is not q.dtype or not out.is_contiguous():
        raise KernelError("out must be contiguous and of q's shape and type")
    if out.data_ptr() & 15:
        raise KernelError("out must start on 16 bytes")
    return out


@functools.lru_cache(maxsize=4096)
def _workspace(*sizes: int) -> int:
    """Bytes that a call of these sizes needs besides its operands."""
    *head, ragged, sequences, rows, window, sinks, longest = sizes
    return library().ivonar_cache_attention_work(*head, 1 if ragged else None, sequences, rows, window, sinks, longest)


def cache_attention(q: Tensor, pages: Tensor, table: Tensor, lengths: Tensor, offsets: Tensor | None = None,
                    window: int = 0, sinks: int = 0, scale: float | None = None, max_length: int | None = None,
                    out: Tensor | None = None) -> Tensor:
    """Attention of q [rows, heads, head_dim] (fp32, fp16 or bfloat16) over the cache, in q's type.

    lengths[b] counts sequence b's cached tokens; the rows of sequence b in q are its last ones, each sees the
    positions up to its own, and with a window (0: none) only the last `window` of them and the first `sinks` of the
    sequence.  heads is a multiple of the cache's kv_heads: head h reads key/value head h // (heads / kv_heads).  A row
    that sees nothing is zero.  scale (default head_dim ** -0.5) multiplies q . k.  max_length, about the longest
    length, sets how keys are shared between blocks (default: what the table can hold); any value gives the same
    result up to the order of sums.  That sharing goes by the average rows of a sequence: single rows over very long
    sequences and chunks of many rows are faster as two calls than as one."""
    device = _device(q, pages, table, lengths, offsets, out)
    count, kv_heads, tiles, dim, sequences, width = _geometry(pages, table, "cache_attention")
    rows, heads, q_row, q_head = _rows(q, None, dim, "q")
    if heads == 0 or heads % kv_heads:
        raise KernelError(f"{heads} heads do not share {kv_heads} key/value heads")
    if rows * (heads // kv_heads) > 1 << 30:
        raise KernelError("too many rows for one call")
    _offsets(offsets, sequences, rows)
    _index(lengths, sequences, "lengths")
    scale = _scale(scale, dim, window, sinks)
    out = _output(q, out)
    if rows == 0:
        return out
    capacity = width * tiles * TOKENS_PER_TILE
    longest = capacity if max_length is None else max(1, min(int(max_length), capacity))
    window, sinks = min(window, 1 << 30), min(sinks, 1 << 30)
    dtype = _DTYPES[q.dtype]
    need = _workspace(dtype, heads, kv_heads, dim, offsets is not None, sequences, rows, window, sinks, longest)
    work = pages.new_empty(need) if need > 0 else None
    _run("ivonar_cache_attention", device, q.data_ptr(), dtype, q_row, q_head, heads, rows, pages.data_ptr(), count,
         kv_heads, tiles, dim, table.data_ptr(), width, lengths.data_ptr(), _address(offsets), sequences, window, sinks,
         scale, longest, out.data_ptr(), _address(work), need)
    return out


def window_attention(q: Tensor, k: Tensor, v: Tensor, offsets: Tensor | None = None, window: int = 0, sinks: int = 0,
                     scale: float | None = None, out: Tensor | None = None) -> Tensor:
    """Causal attention within packed sequences: q [rows, heads, head_dim], k and v [rows, kv_heads, head_dim], all
    fp16 or all bfloat16, in that type.

    offsets (int32 [sequences + 1]): the rows before each sequence; None: all rows are one sequence.  A row sees its
    sequence's rows up to its own, and with a window (0: none) only the last `window` of them and the first `sinks`
    of the sequence.  heads is a multiple of kv_heads.  scale (default head_dim ** -0.5) multiplies q . k.  The
    softmax's weights are rounded to that type for their product with v (their sum is fp32), which adds about as much
    error as the rounding of the result.  Rows that do not start on 16 bytes are copied first."""
    device = _device(q, k, v, offsets, out)
    rows, heads, q_row, q_head = _rows(q, None, None, "q")
    dim = q.shape[2]
    if dim not in HEAD_DIMS:
        raise KernelError(f"head_dim {dim} is not one of {HEAD_DIMS}")
    k_rows, kv_heads, k_row, k_head = _rows(k, None, dim, "k")
    v_rows, _, v_row, v_head = _rows(v, kv_heads, dim, "v")
    if k_rows != rows or v_rows != rows:
        raise KernelError("q, k and v must have the same rows")
    dtype = q.dtype
    if dtype is torch.float32 or k.dtype is not dtype or v.dtype is not dtype:
        raise KernelError("q, k and v must all be float16 or all bfloat16")
    if heads == 0 or kv_heads == 0 or heads % kv_heads:
        raise KernelError(f"{heads} heads do not share {kv_heads} key/value heads")
    if rows * (heads // kv_heads) > 1 << 30 or kv_heads > 65535:
        raise KernelError("too many rows or heads for one call")
    sequences = 1
    if offsets is not None:
        sequences = offsets.shape[0] - 1 if offsets.dim() == 1 else -1
        _index(offsets, max(sequences, 0) + 1, "offsets")
    scale = _scale(scale, dim, window, sinks)
    out = _output(q, out)
    if rows == 0:
        return out
    if ((q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15 or (q_row | q_head | k_row | k_head | v_row | v_head) & 7
            or not dim <= k_row < 1 << 23 or not dim <= v_row < 1 << 23):
        q, k, v = (x.clone(memory_format=torch.contiguous_format) for x in (q, k, v))
        (q_row, q_head, _), (k_row, k_head, _), (v_row, v_head, _) = q.stride(), k.stride(), v.stride()
    _run("ivonar_window_attention", device, q.data_ptr(), k.data_ptr(), v.data_ptr(), _DTYPES[dtype], q_row, q_head,
         k_row, k_head, v_row, v_head, heads, kv_heads, dim, rows, _address(offsets), sequences, min(window, 1 << 30),
         min(sinks, 1 << 30), scale, out.data_ptr())
    return out
