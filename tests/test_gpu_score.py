"""Log probabilities, entropy and alternatives against the definition in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
TYPES = ["float32", "float16", "bfloat16"]


def expected(logits, tokens, temperature):
    """(log probabilities of all logits, of the tokens, entropy, and the bounds of the latter two and of the former).

    Errors: z = (x - m) / T has three roundings of its size; a weight e^z that relative error and 2^-22 of its own; a
    thread adds at most V / 64 of them and the sums then go through fewer than 64 additions; the logarithm and the last
    difference 2^-22 and a rounding of the result's size."""
    x = np.asarray(logits, dtype=np.float64)
    unit = 2.0 ** -24
    z = (x - x.max(1, keepdims=True)) / temperature
    with np.errstate(divide="ignore", invalid="ignore"):
        weights = np.exp(z)
        total = weights.sum(1, keepdims=True)
        p = weights / total
        logs = z - np.log(total)
        finite = np.where(p > 0, z, 0.0)
        entropy = np.log(total[:, 0]) - (p * finite).sum(1)
    size, square = (p * np.abs(finite)).sum(1), (p * finite ** 2).sum(1)
    adding = (x.shape[1] / 64 + 64) * unit
    of_sum = 3 * unit * size + 2.0 ** -22 + adding
    log_total = np.abs(np.log(total[:, 0]))
    of_log = of_sum + 2.0 ** -22 * (1 + log_total)
    bound = 4 * unit * np.abs(np.where(np.isfinite(z), z, 0.0)) + of_log[:, None]
    of_entropy = of_log + 3 * unit * square + size * (2.0 ** -21 + 2 * adding + of_sum) + 2 * unit * size
    rows = np.arange(x.shape[0])
    inside = (tokens >= 0) & (tokens < x.shape[1])
    at = np.where(inside, tokens, 0)
    return logs, np.where(inside, logs[rows, at], -np.inf), entropy, bound, of_entropy


def check(result, logits, tokens, top, temperature, what=""):
    x = logits.double().cpu().numpy()
    t = tokens.cpu().numpy()
    logs, chosen, entropy, bound, of_entropy = expected(x, t, temperature)
    rows = np.arange(x.shape[0])
    got = [r.cpu().numpy() for r in result]

    def close(a, b, limit, name):
        b = np.where(b < -3.4028236e38, -np.inf, b)  # what fp32 makes of numbers past its range
        same = (a == b) | (np.abs(a - b) <= limit)
        assert same.all(), (f"{what} {name}: {int((~same).sum())} off, first at {np.argwhere(~same)[0]}: "
                            f"{a[~same][0]!r} vs {b[~same][0]!r} within {np.broadcast_to(limit, a.shape)[~same][0]:.3g}")

    with np.errstate(invalid="ignore"):
        close(got[0].astype(np.float64), chosen, bound[rows, np.clip(t, 0, x.shape[1] - 1)], "log probability")
        close(got[1].astype(np.float64), entropy, of_entropy, "entropy")
        order = np.argsort(-x, axis=1, kind="stable")[:, :top]
        assert got[2].shape == got[3].shape == (x.shape[0], top)
        assert np.array_equal(got[3], order), f"{what} tokens: first in row {np.argwhere((got[3] != order).any(1))[0]}"
        close(got[2].astype(np.float64), np.take_along_axis(logs, order, 1), np.take_along_axis(bound, order, 1),
              "alternatives")


def _logits(rows, vocab, dtype, seed, spread=3.0):
    import torch

    generator = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, vocab, generator=generator) * spread).to(getattr(torch, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 2, 2), (5, 63, 20), (2, 64, 64), (4, 65, 64), (7, 2047, 5),
                                            (2, 2048, 0), (3, 2049, 33), (1, 32000, 20), (6, 32001, 64), (2, 100003, 20),
                                            (1, 262144, 64), (1100, 300, 7), (1500, 4095, 20), (1030, 4100, 20)])
def test_against_the_definition(cuda, dtype, rows, vocab, top):
    """One row and many, a wave or a block for a row or several blocks, widths around the chunks; tied halves."""
    import torch
    from ivonar_amd import sampling

    logits = _logits(rows, vocab, dtype, rows + vocab).to(cuda)
    tokens = torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(1)).to(cuda)
    for temperature in (1.0, 0.3):
        check(sampling.log_probabilities(logits, tokens, top, temperature), logits, tokens, top, temperature)


@pytest.mark.parametrize("dtype", TYPES)
def test_orders_that_move_the_bound(cuda, dtype):
    """Rising, falling and equal logits, a few distinct values, and the largest ones all in one lane's places."""
    import torch
    from ivonar_amd import sampling

    vocab = 9001
    ramp = torch.linspace(-20, 20, vocab)
    rows = [ramp, ramp.flip(0), torch.zeros(vocab), torch.full((vocab,), -3.0), (torch.arange(vocab) % 3).float(),
            (torch.arange(vocab) % 2048 < 8).float() * 5 - ramp * 1e-2, (torch.arange(vocab) % 256 == 7).float()]
    logits = torch.stack(rows).to(getattr(torch, dtype)).to(cuda)
    tokens = torch.arange(len(rows), device=cuda) * 1000
    for top in (1, 20, 64):
        check(sampling.log_probabilities(logits, tokens, top), logits, tokens, top, 1.0, f"top {top}")
    many = logits.repeat(200, 1)[:, :4000].contiguous()  # a wave for a row
    check(sampling.log_probabilities(many, tokens.repeat(200), 20), many, tokens.repeat(200), 20, 1.0, "many")


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_logits(cuda, dtype):
    """-inf and the type's lowest value in most places, in all of them, and a single logit left."""
    import torch
    from ivonar_amd import sampling

    kind = getattr(torch, dtype)
    vocab, top = 5000, 20
    logits = _logits(8, vocab, dtype, 5)
    lowest = torch.finfo(kind).min
    logits[0, 10:] = -float("inf")
    logits[1, :-3] = -float("inf")
    logits[2] = -float("inf")
    logits[3, 10:] = lowest
    logits[4] = lowest
    logits[5] = -float("inf")
    logits[5, 777] = 1.5
    logits[6] = torch.finfo(kind).max
    logits[7] = lowest
    logits[7, 4321] = torch.finfo(kind).max
    logits = logits.to(cuda)
    tokens = torch.tensor([3, 4999, 0, 12, 4999, 777, 2, 4321], device=cuda)
    got = sampling.log_probabilities(logits, tokens, top)
    some = [0, 1, 3, 4, 5, 6, 7]
    check([r[some] for r in got], logits[some], tokens[some], top, 1.0)
    assert got.log_probability[2] == -float("inf") and got.entropy[2] == 0
    assert got.top_token[2].tolist() == list(range(top)) and (got.top_log_probability[2] == -float("inf")).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_not_numbers(cuda, dtype):
    """A NaN or +inf makes its own row's numbers NaN and no other's; NaN is listed behind every number."""
    import torch
    from ivonar_amd import sampling

    logits = _logits(6, 3000, dtype, 6)
    logits[1, 2999] = float("nan")
    logits[3, 5] = float("inf")
    logits[4] = float("nan")
    logits[4, 100:102] = torch.tensor([1.0, 2.0])
    logits = logits.to(cuda)
    tokens = torch.zeros(6, dtype=torch.int64, device=cuda)
    got = sampling.log_probabilities(logits, tokens, 4)
    for row in range(6):
        odd = row in (1, 3, 4)
        assert torch.isnan(got.log_probability[row]) == odd and torch.isnan(got.entropy[row]) == odd
        assert torch.isnan(got.top_log_probability[row]).all() == odd
    check([r[[0, 2, 5]] for r in got], logits[[0, 2, 5]], tokens[:3], 4, 1.0)
    best = torch.sort(logits[1, :2999].float(), descending=True, stable=True).indices[:4]
    assert torch.equal(got.top_token[1], best)
    assert got.top_token[3, 0] == 5
    assert got.top_token[4].tolist() == [101, 100, 0, 1]


def test_tokens_outside_and_signed_zeros(cuda):
    import torch
    from ivonar_amd import sampling

    logits = torch.zeros(4, 100, device=cuda)
    logits[:, ::2] = -0.0
    tokens = torch.tensor([-1, 100, -100, 2 ** 40], device=cuda)
    got = sampling.log_probabilities(logits, tokens, 3)
    assert (got.log_probability == -float("inf")).all()
    assert got.top_token.tolist() == [[0, 1, 2]] * 4
    assert torch.allclose(got.entropy, torch.full((4,), float(np.log(100)), device=cuda))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lead", [0, 1, 2, 3, 5, 7])
def test_rows_off_alignment(cuda, dtype, lead):
    """Rows of an odd stride that start anywhere; what lies before and behind them is not seen."""
    import torch
    from ivonar_amd import sampling

    rows, vocab = 5, 2051
    whole = torch.full((rows, vocab + 12), 1e4, dtype=getattr(torch, dtype), device=cuda)
    whole[:, lead:lead + vocab] = _logits(rows, vocab, dtype, lead).to(cuda)
    logits = whole[:, lead:lead + vocab]
    tokens = torch.arange(rows, device=cuda) * 400
    check(sampling.log_probabilities(logits, tokens, 20), logits, tokens, 20, 1.0)
    odd = torch.cat([whole.flatten(), whole.new_zeros(3)])[:rows * (vocab + 11)].view(rows, vocab + 11)
    logits = odd[:, lead:lead + vocab]
    check(sampling.log_probabilities(logits, tokens, 20), logits, tokens, 20, 1.0)


def test_past_32_bits(cuda):
    """Logits that lie more than 2^31 elements into their tensor."""
    import torch
    from ivonar_amd import sampling

    rows, vocab = 70000, 32000
    logits = torch.zeros(rows, vocab, dtype=torch.float16, device=cuda)  # 4.5 GB
    tail = _logits(3, vocab, "float16", 9).to(cuda)
    logits[-3:] = tail
    tokens = torch.full((rows,), 17, dtype=torch.int64, device=cuda)
    got = sampling.log_probabilities(logits, tokens, 5)
    check([r[-3:] for r in got], tail, tokens[-3:], 5, 1.0)
    assert torch.allclose(got.entropy[:-3], torch.full((), float(np.log(vocab)), device=cuda), atol=1e-4)
    assert (got.top_token[:-3] == torch.arange(5, device=cuda)).all()


def test_streams_and_graphs(cuda):
    """Two calls at once on two streams, and a captured one replayed with other logits in place."""
    import torch
    from ivonar_amd import sampling

    a, b = _logits(2, 32000, "float32", 1).to(cuda), _logits(700, 5000, "bfloat16", 2).to(cuda)
    ta, tb = torch.tensor([5, 7], device=cuda), torch.arange(700, device=cuda)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for _ in range(3):
        for stream, logits, tokens in zip(streams, (a, b), (ta, tb)):
            with torch.cuda.stream(stream):
                results.append(sampling.log_probabilities(logits, tokens, 20))
    torch.cuda.synchronize()
    for i, got in enumerate(results):
        check(got, (a, b)[i % 2], (ta, tb)[i % 2], 20, 1.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sampling.log_probabilities(a, ta, 20, 0.8)
    for replay in range(4):
        a.copy_(_logits(2, 32000, "float32", 50 + replay))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check(got, a, ta, 20, 0.8, f"replay {replay}")


def test_refusals(cuda):
    import torch
    from ivonar_amd import sampling
    from ivonar_amd.runtime import KernelError

    logits, tokens = torch.zeros(4, 100, device=cuda), torch.zeros(4, dtype=torch.int64, device=cuda)
    good = dict(logits=logits, tokens=tokens, top=5, temperature=1.0)
    sampling.log_probabilities(**good)
    for name, value in (("logits", logits[0]), ("logits", logits.double()), ("logits", logits.t()[:4]),
                        ("logits", logits[:, :0]), ("logits", logits.cpu()), ("logits", logits[:3]),
                        ("tokens", tokens.int()), ("tokens", tokens[:3]), ("tokens", tokens[:, None]),
                        ("tokens", tokens.cpu()), ("top", -1), ("top", 65), ("temperature", 0.0), ("temperature", -1.0),
                        ("temperature", float("nan")), ("temperature", float("inf")), ("temperature", 1e-40)):
        with pytest.raises(KernelError):
            sampling.log_probabilities(**{**good, name: value})
    with pytest.raises(KernelError):
        sampling.log_probabilities(logits[:, :4].contiguous(), tokens, 5)
    with pytest.raises(KernelError):
        sampling.log_probabilities(logits[:1, :1].expand(1 << 31, 1), tokens)
    empty = sampling.log_probabilities(logits[:0], tokens[:0], 5)
    assert [tuple(r.shape) for r in empty] == [(0,), (0,), (0, 5), (0, 5)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_rows_past_32_bits(cuda, dtype):
    """Rows that lie 4 GiB and more apart."""
    import torch
    from ivonar_amd import sampling

    vocab, apart = 5003, (1 << 32) // (4 if dtype == "float32" else 2) + 12345
    flat = torch.empty(2 * apart + vocab, dtype=getattr(torch, dtype), device=cuda)
    logits = flat.as_strided((3, vocab), (apart, 1))
    logits.copy_(torch.randn(3, vocab, generator=torch.Generator().manual_seed(1)))
    tokens = torch.tensor([0, 5002, 77], device=cuda)
    check(sampling.log_probabilities(logits, tokens, 9), logits.clone(), tokens, 9, 1.0)
