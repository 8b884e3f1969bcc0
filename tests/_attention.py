"""A plain 64-bit implementation of the 4-bit cache and of attention with a window and sinks, and the bounds that the
kernels' results keep against it."""

from __future__ import annotations

import math

import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
# bf16 terms that a row's values and weights are split into, and the unit of the results' type
TERMS = {"float32": 3, "float16": 2, "bfloat16": 1}
UNIT = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def block_exponent(most: np.ndarray) -> np.ndarray:
    """floor(log2(most * 8/7)) - 2 within -100 .. 125, by comparing with powers of two."""
    exponent = np.full(most.shape, -100)
    for e in range(-99, 126):
        exponent[most >= 1.75 * 2.0 ** (e + 1)] = e
    return exponent


def stored(x: np.ndarray) -> np.ndarray:
    """What the cache gives back for rows x [..., dim]: the nearest value of the block's grid, ties to the even code."""
    blocks = np.asarray(x, dtype=np.float64).reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    finite = np.isfinite(blocks).all(-1, keepdims=True)
    blocks = np.where(finite, blocks, 0.0)
    step = 2.0 ** block_exponent(np.abs(blocks).max(-1, keepdims=True))
    y = np.abs(blocks) / step
    code = np.zeros(y.shape, dtype=int)
    for c in range(1, 8):
        middle = (GRID[c - 1] + GRID[c]) / 2
        code += (y >= middle) if c % 2 == 0 else (y > middle)
    value = np.copysign(GRID[code] * step, blocks)
    return np.where(finite, value, np.nan).reshape(x.shape)


def visible(position: int, keys: int, window: int, sinks: int) -> np.ndarray:
    key = np.arange(keys)
    seen = key <= position
    if window:
        seen &= (key > position - window) | (key < sinks)
    return seen


def attend(q, k, v, first, window=0, sinks=0, scale=None, missing=None):
    """(out, spread, size) of q [n, heads, dim] at positions first .. over k, v [keys, kv_heads, dim]: the attention,
    sum p |v| (what an error of the weights can move), and the largest sum |q| |k| scale that a row's logits have.
    missing [keys]: keys that nobody sees."""
    q, k, v = (np.asarray(x, dtype=np.float64) for x in (q, k, v))
    n, heads, dim = q.shape
    group = heads // k.shape[1]
    scale = dim ** -0.5 if scale is None else scale
    out, spread, size = np.zeros_like(q), np.zeros_like(q), np.zeros((n, heads, 1))
    for i in range(n):
        seen = visible(first + i, k.shape[0], window, sinks)
        if missing is not None:
            seen &= ~missing
        if not seen.any():
            continue
        for h in range(heads):
            keys, values = k[seen, h // group], v[seen, h // group]
            logits = keys @ q[i, h] * scale
            size[i, h] = (np.abs(keys) @ np.abs(q[i, h])).max() * scale
            p = np.exp(logits - logits.max())
            p /= p.sum()
            out[i, h], spread[i, h] = p @ values, p @ np.abs(values)
    return out, spread, size


def bound(out, spread, size, dtype: str, keys: int, dim: int, weight_unit: float | None = None):
    """How far a result in `dtype` may be from `out`.

    Logits: products of exact operands summed in fp32, dim of them with up to three terms each, then scaled and
    shifted: (3 dim + 8) 2^-24 of `size`, which is a relative error of each weight; the exponential adds 2^-22.
    Weights: rounded for the product with the values, not for their sum, with an error of weight_unit; by default what
    TERMS[dtype] bf16 terms (8 bits each) leave, more than the cache attention's two terms for bfloat16 rows.  Sums over
    the keys: keys + 64 roundings of 2^-24 each, in numerator and denominator.  Last, the rounding to the result's type."""
    if weight_unit is None:
        weight_unit = max(2.0 ** (-8 * TERMS[dtype] - 1), 2.0 ** -24)
    relative = weight_unit + 2 * ((3 * dim + 8) * 2.0 ** -24 * size + 2.0 ** -22) + 2 * (keys + 64) * 2.0 ** -24
    return relative * spread + UNIT[dtype] * np.abs(out) + 1e-30


def check(actual, expected, spread, size, dtype: str, keys: int, dim: int, what: str = "", **more):
    actual = np.asarray(actual, dtype=np.float64)
    far = np.abs(actual - expected)
    limit = bound(expected, spread, size, dtype, keys, dim, **more)
    bad = ~(far <= limit)
    if bad.any():
        index = tuple(np.argwhere(bad)[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.size} off; first at {index}: {actual[index]!r} vs "
                             f"{expected[index]!r}, {far[index]:.3g} > {limit[index]:.3g}")


def place(lengths, page_size: int, rng, spare: int = 3, width: int = 1):
    """A page table for sequences of these lengths: (pages, table int32), pages scattered, unused entries -1."""
    needed = [math.ceil(n / page_size) for n in lengths]
    total = sum(needed) + spare
    order = rng.permutation(total)
    table = np.full((len(lengths), max(needed) + width), -1, dtype=np.int32)
    start = 0
    for row, count in enumerate(needed):
        table[row, :count] = order[start:start + count]
        start += count
    return total, table


def cancelling(length: int, dim: int):
    """(k, v, scale) of keys that the cache holds exactly, for q = (1, 0, ..): every third one has the weight 1 and the
    others 0.5 + 0.4 / 256, which bfloat16 rounds to 0.5, and values whose weighted sum is small against their size."""
    third = np.arange(length) % 3 == 2
    k = np.zeros((length, 1, dim), np.float32)
    k[third, :, 0] = 1
    v = np.resize(np.float32([6, -4, 3, 2, -1.5, 1, -0.5, 6]), (length, 1, dim)).copy()
    v[third] *= -1
    return k, v, -math.log(0.5 + 0.4 / 256)
