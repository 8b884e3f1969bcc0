"""Log probabilities where the largest logit over the temperature is past what fp32 holds to a fraction of one: masks by
large numbers, low and high temperatures, large logits."""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
TYPES = ["float32", "float16", "bfloat16"]
UNIT = 2.0 ** -24
EDGE = 11629080.0  # 2^24 ln 2: the logit whose share of log2(e) is 2^24


def expected(logits, tokens, temperature):
    """(log probabilities of all logits, of the tokens, entropy, and the bounds of the three).

    Errors: log2(e) / T has three roundings, and a z one or two more: five of z's size, whichever way it is formed, and
    two for the way back to nats and one for the last difference, eight in a log probability.  A weight has its z's and
    2^-22 of its own, and as much again each time that its sum moves to another maximum: at most once per chunk and eight
    times in the joins.  A thread adds at most V / 64 weights, and their sums go through fewer than 64 additions."""
    x = np.asarray(logits, dtype=np.float64)
    moves = x.shape[1] / 2048 + 9
    with np.errstate(divide="ignore", invalid="ignore", under="ignore"):
        z = (x - x.max(1, keepdims=True)) / temperature
        weights = np.exp(z)
        total = weights.sum(1, keepdims=True)
        p = weights / total
        logs = z - np.log(total)
        finite = np.where(p > 0, z, 0.0)
    log_total = np.log(total[:, 0])
    size, square = (p * np.abs(finite)).sum(1), (p * finite ** 2).sum(1)
    of_sum = 5 * UNIT * size + moves * 2.0 ** -22 + (x.shape[1] / 64 + 64) * UNIT
    of_total = of_sum + 2.0 ** -22 * (1 + np.abs(log_total))
    bound = 8 * UNIT * np.abs(np.where(np.isfinite(z), z, 0.0)) + of_total[:, None]
    of_entropy = of_total + 5 * UNIT * square + size * (2 * of_sum + 4 * UNIT)
    entropy = log_total - (p * finite).sum(1)
    rows = np.arange(x.shape[0])
    return logs, logs[rows, tokens], entropy, bound, of_entropy


def check(result, logits, tokens, top, temperature, what):
    x, t = logits.double().cpu().numpy(), tokens.cpu().numpy()
    logs, chosen, entropy, bound, of_entropy = expected(x, t, temperature)
    rows = np.arange(x.shape[0])
    got = [r.double().cpu().numpy() for r in result]

    def close(a, b, limit, name):
        b = np.where(b < -3.4028235e38, -np.inf, b)  # past fp32's range
        with np.errstate(invalid="ignore"):
            same = (a == b) | (np.abs(a - b) <= limit)
        assert same.all(), (f"{what} {name}: {int((~same).sum())} off, first at {np.argwhere(~same)[0]}: "
                            f"{a[~same][0]!r} vs {b[~same][0]!r} within {np.broadcast_to(limit, a.shape)[~same][0]:.3g}")

    close(got[0], chosen, bound[rows, t], "log probability")
    close(got[1], entropy, of_entropy, "entropy")
    order = np.argsort(-x, axis=1, kind="stable")[:, :top]
    assert np.array_equal(got[3], order), what
    close(got[2], np.take_along_axis(logs, order, 1), np.take_along_axis(bound, order, 1), f"{what} alternatives")


def _check_call(logits, temperature, what, repeats=1):
    """The call on these rows, and on many copies of them, by one wave each."""
    import torch
    from ivonar_amd import sampling

    temperature = float(np.float32(temperature))  # as the kernel takes it
    rows, vocab = logits.shape
    tokens = torch.stack([logits.argmax(1), torch.full((rows,), 3, device=logits.device)])[torch.arange(rows) % 2,
                                                                                       torch.arange(rows)]
    top = min(20, vocab)
    if repeats > 1:
        many = sampling.log_probabilities(logits.repeat(repeats, 1), tokens.repeat(repeats), top, temperature)
        for values in many:
            values = values.view(repeats, rows, -1)
            assert (values == values[:1]).all() or torch.isnan(values).any(), what
        got = [values[:rows] for values in many]
    else:
        got = sampling.log_probabilities(logits, tokens, top, temperature)
    check(got, logits, tokens, top, temperature, what)


def _logits(rows, vocab, dtype, seed, spread=3.0):
    import torch

    generator = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, vocab, generator=generator) * spread).to(getattr(torch, dtype))


SHAPES = [(3, 5000, 1), (2, 32000, 1), (1, 262144, 1), (2, 5000, 2100), (3, 300, 1)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,repeats", SHAPES)
def test_masks_of_large_numbers(cuda, dtype, rows, vocab, repeats):
    """All but a few logits at a number that weighs nothing, in whole lanes' places, with temperatures around one."""
    import torch

    for mask in (-1e4, -6e4) if dtype == "float16" else (-1e4, -1e9, -1e10, -1e20, -1e30, -1e38):
        logits = _logits(rows, vocab, dtype, 5)
        logits[:, 10:] = mask
        logits[-1, :10] = mask
        logits[-1, vocab // 2:vocab // 2 + 9] = _logits(1, 9, dtype, 6)[0]
        for temperature in (1.0, 0.7, 0.3, 1e-4, 3.0):
            _check_call(logits.to(cuda), temperature, f"mask {mask} at {temperature}", repeats)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,repeats", SHAPES)
def test_low_and_high_temperatures(cuda, dtype, rows, vocab, repeats):
    logits = _logits(rows, vocab, dtype, 8)
    logits[0, 1] = logits[0].max()  # two that share the row at the lowest temperatures
    logits[-1] -= 40.0
    logits = logits.to(cuda)
    for temperature in (1e-3, 1e-6, 1e-7, 1e-8, 1e-9, 1e-12, 1e-30, 2.1e-38, 1e4, 1e30, 9e37):
        _check_call(logits, temperature, f"temperature {temperature}", repeats)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,vocab,repeats", SHAPES)
def test_large_logits(cuda, dtype, rows, vocab, repeats):
    """Logits of all sizes, at temperatures of their size and far below and above it, of either sign."""
    for size in (1e6, 1e9, 1e15, 1e20, 1e30, 1e37):
        logits = (_logits(rows, vocab, "float32", 9) * size).to(_logits(1, 1, dtype, 0).dtype)
        logits[-1] -= 8 * size
        for temperature in (1.0, 1e-3 * size, size, 2 * size, 100 * size):
            if temperature < 1e38:
                _check_call(logits.to(cuda), temperature, f"size {size} at {temperature}", repeats)


@pytest.mark.parametrize("rows,vocab,repeats", SHAPES)
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_maxima_on_both_sides_of_the_edge(cuda, rows, vocab, repeats, sign):
    """Maxima whose product with log2(e) / T lies just below 2^24 in some lanes and just above it in others."""
    import torch

    generator = torch.Generator().manual_seed(10)
    for spread in (4, 60, 5000):
        logits = sign * EDGE + torch.randint(-spread, spread + 1, (rows, vocab), generator=generator).float()
        for temperature in (1.0, 1.0000002, 0.9999999, 0.5, 2.0):
            _check_call(logits.to(cuda), temperature, f"within {spread} at {temperature}", repeats)
    rising = (sign * EDGE + torch.arange(vocab).float() / vocab * 80 - 40).expand(rows, vocab).contiguous()
    _check_call(rising.to(cuda), 1.0, "rising", repeats)
    _check_call(rising.flip(1).contiguous().to(cuda), 1.0, "falling", repeats)


def test_differences_past_the_range(cuda):
    """Logits whose difference is no fp32 number while the log probability is one, or is past the range itself."""
    import torch

    big = torch.finfo(torch.float32).max
    logits = _logits(2, 3000, "float32", 11) * 1e37
    logits[:, 3], logits[:, 2000] = -big, big
    logits[1] = torch.where(torch.arange(3000) % 3 == 0, -big, big)
    for temperature in (1.0, 1e20, 1e30, 1e37, 9e37):
        _check_call(logits.to(cuda), temperature, f"temperature {temperature}")
