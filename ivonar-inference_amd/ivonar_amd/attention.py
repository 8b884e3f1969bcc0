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
instance) is no page: nothing is written there, zeros are read, and attention does not see its tokens, so pages
before a window may be handed back.  ``offsets`` (int32 [sequences + 1]) are the rows before each sequence in a ragged
batch; None stands for one row per sequence.  Rows past the last sequence's (padding) are not written to the cache,
and are zero in the results.  Index tensors stay on the device: no call reads them on the host, allocates more than
its results and a workspace, or synchronises, so all of them can be captured into a graph.
"""

from __future__ import annotations

import math

import torch
from torch import Tensor

from .ops import _address, _call, _require_device
from .runtime import KernelError, library

TOKENS_PER_TILE = 32
HEAD_DIMS = (64, 128, 256)
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


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


def _geometry(pages: Tensor, table: Tensor, what: str) -> tuple[int, int, int, int]:
    """(pages, kv_heads, tiles per page, head_dim) of a cache, with its table checked."""
    if pages.dtype != torch.uint8 or pages.ndim != 4 or not pages.is_contiguous():
        raise KernelError(f"{what} needs pages as cache_pages() makes them")
    count, heads, tiles, size = pages.shape
    if size % 34 or size // 34 not in HEAD_DIMS or tiles & (tiles - 1) or pages.numel() == 0:
        raise KernelError(f"{what} needs pages as cache_pages() makes them")
    if table.dtype != torch.int32 or table.ndim != 2 or not table.is_contiguous():
        raise KernelError(f"{what} needs a contiguous int32 table [sequences, width]")
    if table.shape[1] * tiles * TOKENS_PER_TILE > 1 << 30:
        raise KernelError(f"{what}: a sequence has at most 2**30 tokens")
    return count, heads, tiles, size // 34


def _index(tensor: Tensor, count: int, device: torch.device, what: str) -> None:
    if (tensor.dtype != torch.int32 or tensor.ndim != 1 or tensor.shape[0] != count or not tensor.is_contiguous()
            or tensor.device != device):
        raise KernelError(f"{what} must be contiguous int32 [{count}] on the cache's device")


def _sequences(table: Tensor, offsets: Tensor | None, rows: int, device: torch.device) -> int:
    sequences = table.shape[0]
    if offsets is not None:
        _index(offsets, sequences + 1, device, "offsets")
    elif rows != sequences:
        raise KernelError(f"{rows} rows of {sequences} sequences need offsets")
    return sequences


def _rows(x: Tensor, heads: int | None, head_dim: int | None, device: torch.device, what: str) -> int:
    if x.ndim != 3 or (heads is not None and x.shape[1] != heads) or (head_dim is not None and x.shape[2] != head_dim):
        raise KernelError(f"{what} must be [rows, {heads or 'heads'}, {head_dim or 'head_dim'}], not {list(x.shape)}")
    if x.dtype not in _DTYPES:
        raise KernelError(f"{what} must be float32, float16 or bfloat16, not {x.dtype}")
    if x.stride(2) != 1 or x.device != device:
        raise KernelError(f"{what} must have a head's values side by side, on the device of the other tensors")
    return x.shape[0]


def _same_device(device: torch.device, *tensors: Tensor) -> None:
    if any(tensor.device != device for tensor in tensors):
        raise KernelError("the tensors of a call must be on one device")


def cache_write(pages: Tensor, k: Tensor, v: Tensor, table: Tensor, past: Tensor, offsets: Tensor | None = None) -> None:
    """Quantises rows of k and v [rows, kv_heads, head_dim] (fp32, fp16 or bfloat16, any row and head stride) into the
    cache: row r of sequence b becomes position past[b] + r - offsets[b]."""
    device = _require_device(pages, k, v, table, past, offsets)
    count, heads, tiles, dim = _geometry(pages, table, "cache_write")
    rows = _rows(k, heads, dim, device, "k")
    if _rows(v, heads, dim, device, "v") != rows or v.dtype != k.dtype:
        raise KernelError("k and v must have the same rows and type")
    _same_device(device, pages, table)
    sequences = _sequences(table, offsets, rows, device)
    _index(past, sequences, device, "past")
    if rows == 0:
        return
    _call("ivonar_cache_write", device, k.data_ptr(), v.data_ptr(), _DTYPES[k.dtype], k.stride(0), k.stride(1),
          v.stride(0), v.stride(1), rows, pages.data_ptr(), count, heads, tiles, dim, table.data_ptr(), table.shape[1],
          past.data_ptr(), _address(offsets), sequences)


def cache_read(pages: Tensor, table: Tensor, start: Tensor | None, offsets: Tensor | None, rows: int,
               dtype: torch.dtype = torch.float32) -> tuple[Tensor, Tensor]:
    """(k, v) [rows, kv_heads, head_dim] as `dtype`: row r of sequence b is position start[b] + r - offsets[b] (start
    None: 0)."""
    device = _require_device(pages, table, start, offsets)
    count, heads, tiles, dim = _geometry(pages, table, "cache_read")
    _same_device(device, pages, table)
    if dtype not in _DTYPES:
        raise KernelError(f"the cache is read as float32, float16 or bfloat16, not {dtype}")
    if rows < 0:
        raise KernelError("rows must not be negative")
    sequences = _sequences(table, offsets, rows, device)
    if start is not None:
        _index(start, sequences, device, "start")
    k, v = torch.empty((2, rows, heads, dim), dtype=dtype, device=device)
    if rows:
        _call("ivonar_cache_read", device, pages.data_ptr(), count, heads, tiles, dim, table.data_ptr(), table.shape[1],
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
        return torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or not out.is_contiguous():
        raise KernelError("out must be contiguous and of q's shape, type and device")
    return out


def cache_attention(q: Tensor, pages: Tensor, table: Tensor, lengths: Tensor, offsets: Tensor | None = None,
                    window: int = 0, sinks: int = 0, scale: float | None = None, max_length: int | None = None,
                    out: Tensor | None = None) -> Tensor:
    """Attention of q [rows, heads, head_dim] (fp32, fp16 or bfloat16) over the cache, in q's type.

    lengths[b] counts sequence b's cached tokens; the rows of sequence b in q are its last ones, each sees the
    positions up to its own, and with a window (0: none) only the last `window` of them and the first `sinks` of the
    sequence.  heads is a multiple of the cache's kv_heads: head h reads key/value head h // (heads / kv_heads).  A row
    that sees nothing is zero.  scale (default head_dim ** -0.5) multiplies q . k.  max_length, about the longest
    length, sets how keys are shared between blocks (default: what the table can hold); any value gives the same
    result up to the order of sums."""
    device = _require_device(q, pages, table, lengths, offsets)
    count, kv_heads, tiles, dim = _geometry(pages, table, "cache_attention")
    rows = _rows(q, None, dim, device, "q")
    heads = q.shape[1]
    if heads == 0 or heads % kv_heads:
        raise KernelError(f"{heads} heads do not share {kv_heads} key/value heads")
    if rows * (heads // kv_heads) > 1 << 30:
        raise KernelError("too many rows for one call")
    _same_device(device, pages, table)
    sequences = _sequences(table, offsets, rows, device)
    _index(lengths, sequences, device, "lengths")
    scale = _scale(scale, dim, window, sinks)
    out = _output(q, out)
    if rows == 0:
        return out
    capacity = table.shape[1] * tiles * TOKENS_PER_TILE
    longest = capacity if max_length is None else max(1, min(int(max_length), capacity))
    window, sinks = min(window, 1 << 30), min(sinks, 1 << 30)
    dtype, address = _DTYPES[q.dtype], _address(offsets)
    need = library().ivonar_cache_attention_work(dtype, heads, kv_heads, dim, address, sequences, rows, window, sinks,
                                                 longest)
    work = torch.empty(need, dtype=torch.uint8, device=device) if need > 0 else None
    _call("ivonar_cache_attention", device, q.data_ptr(), dtype, q.stride(0), q.stride(1), heads, rows,
          pages.data_ptr(), count, kv_heads, tiles, dim, table.data_ptr(), table.shape[1], lengths.data_ptr(), address,
          sequences, window, sinks, scale, longest, out.data_ptr(), _address(work), max(need, 0))
    return out


def _by_sixteen_bytes(x: Tensor) -> Tensor:
    """x with rows that start on 16 bytes, after a copy where they do not (or lie further apart than a call takes)."""
    if x.data_ptr() % 16 == 0 and x.stride(0) % 8 == 0 and x.stride(1) % 8 == 0 and x.stride(0) < 1 << 23:
        return x
    return x.clone(memory_format=torch.contiguous_format)


def window_attention(q: Tensor, k: Tensor, v: Tensor, offsets: Tensor | None = None, window: int = 0, sinks: int = 0,
                     scale: float | None = None, out: Tensor | None = None) -> Tensor:
    """Causal attention within packed sequences: q [rows, heads, head_dim], k and v [rows, kv_heads, head_dim], all
    fp16 or all bfloat16, in that type.

    offsets (int32 [sequences + 1]): the rows before each sequence; None: all rows are one sequence.  A row sees its
    sequence's rows up to its own, and with a window (0: none) only the last `window` of them and the first `sinks`
    of the sequence.  heads is a multiple of kv_heads.  scale (default head_dim ** -0.5) multiplies q . k.  Rows that
    do not start on 16 bytes are copied first."""
    device = _require_device(q, k, v, offsets)
    dim = q.shape[-1]
    if dim not in HEAD_DIMS:
        raise KernelError(f"head_dim {dim} is not one of {HEAD_DIMS}")
    rows = _rows(q, None, None, device, "q")
    heads, kv_heads = q.shape[1], k.shape[1] if k.ndim == 3 else 0
    if _rows(k, None, dim, device, "k") != rows or _rows(v, kv_heads, dim, device, "v") != rows:
        raise KernelError("q, k and v must have the same rows")
    if q.dtype == torch.float32 or k.dtype != q.dtype or v.dtype != q.dtype:
        raise KernelError("q, k and v must all be float16 or all bfloat16")
    if heads == 0 or kv_heads == 0 or heads % kv_heads:
        raise KernelError(f"{heads} heads do not share {kv_heads} key/value heads")
    if rows * (heads // kv_heads) > 1 << 30 or kv_heads > 65535:
        raise KernelError("too many rows or heads for one call")
    sequences = 1
    if offsets is not None:
        sequences = offsets.shape[0] - 1 if offsets.ndim == 1 else -1
        _index(offsets, max(sequences, 0) + 1, device, "offsets")
    scale = _scale(scale, dim, window, sinks)
    out = _output(q, out)
    if rows == 0:
        return out
    q, k, v = _by_sixteen_bytes(q), _by_sixteen_bytes(k), _by_sixteen_bytes(v)
    _call("ivonar_window_attention", device, q.data_ptr(), k.data_ptr(), v.data_ptr(), _DTYPES[q.dtype], q.stride(0),
          q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1), heads, kv_heads, dim, rows,
          _address(offsets), sequences, min(window, 1 << 30), min(sinks, 1 << 30), scale, out.data_ptr())
    return out
