"""Device sampling state and launches (reference: decoder.py:324-371 sampling rule and
configure_sampling; kernel_decoder.py:213-224 and :619-681 the logit_bounds / sample_token launches).

``DeviceSampler`` owns the buffers the two kernels read and write (temperature, penalty,
inverse_penalty, top_k, seen, bounds, uniform, token), validates the rule on the host as the
reference's ``configure_sampling`` does, and launches both kernels on the current stream.  Nothing
here synchronises except ``sample()``, which returns the token as a Python int.

``log_probabilities(logits, tokens, top, temperature)`` gives the log probabilities of tokens that are
known (a prompt's, or the ones just drawn), the entropy, and the likeliest alternatives (the reference has
no counterpart).
"""

from __future__ import annotations

import functools
from typing import Iterable, NamedTuple

import torch
from torch import Tensor

from .attention import _DTYPES, _device, _run
from .runtime import KernelError, check, current_stream, int32, library, pointer

SAMPLE_THREADS = 1024  # largest top-k one sampling block handles (kernel_decoder.py:25)
BOUND_GROUP = 64       # logits per bound (kernel_decoder.py:26)
MAX_VOCAB = 1 << 18
MAX_TOP = 64           # most alternatives of log_probabilities


class DeviceSampler:
    """Temperature / repetition-penalty / top-k sampling of one sequence on the device."""

    def __init__(self, vocab: int, device: torch.device | str, max_top_k: int = 256) -> None:
        device = torch.device(device)
        if device.type != "cuda":
            raise KernelError("the device sampler needs a ROCm device")
        if not 0 < vocab <= MAX_VOCAB:
            raise KernelError(f"vocab {vocab} outside 1..{MAX_VOCAB}")
        if not 0 < max_top_k <= SAMPLE_THREADS:
            raise KernelError(f"max_top_k {max_top_k} outside 1..{SAMPLE_THREADS}")
        lib = library()
        check(lib.ivonar_define(b"MAX_TOPK", int(max_top_k)), "define MAX_TOPK")
        self.vocab = int(vocab)
        self.max_top_k = int(max_top_k)
        self.device = device
        self.temperature = torch.ones(1, dtype=torch.float32, device=device)
        self.penalty = torch.ones(1, dtype=torch.float32, device=device)
        self.inverse_penalty = torch.ones(1, dtype=torch.float32, device=device)
        self.top_k = torch.ones(1, dtype=torch.int64, device=device)
        self.seen = torch.zeros((1, vocab), dtype=torch.bool, device=device)
        self.bounds = torch.zeros((vocab + BOUND_GROUP - 1) // BOUND_GROUP, dtype=torch.float32, device=device)
        self.uniform = torch.zeros(1, dtype=torch.float32, device=device)
        self.token = torch.zeros(1, dtype=torch.int64, device=device)

    def configure_sampling(self, temperature: float, top_k: int, repetition_penalty: float = 1.0,
                           penalized_ids: Iterable[int] = ()) -> None:
        """The rule of decoder.py:340-361: a non-positive temperature or penalty is a ValueError, a top_k
        outside 1..max_top_k selects max_top_k, and the in-vocabulary ids of `penalized_ids` are marked
        as already generated (the rest are ignored)."""
        if any(value <= 0 for value in (temperature, repetition_penalty)):
            raise ValueError("temperature and repetition_penalty must be positive")
        k = int(top_k)
        if not 1 <= k <= self.max_top_k:
            k = self.max_top_k
        penalty = float(repetition_penalty)
        for buffer, value in ((self.temperature, float(temperature)), (self.penalty, penalty),
                              (self.inverse_penalty, 1.0 / penalty), (self.top_k, k)):
            buffer.fill_(value)
        ids = torch.as_tensor([int(i) for i in penalized_ids], dtype=torch.int64)
        marked = torch.zeros((1, self.vocab), dtype=torch.bool)
        marked[0, ids[(ids >= 0) & (ids < self.vocab)]] = True
        self.seen.copy_(marked)

    def launch(self, logits: Tensor, uniform: Tensor | None = None, token: Tensor | None = None,
               history: Tensor | None = None) -> None:
        """logit_bounds then sample_token on the current stream; draws with `uniform` (default: this
        sampler's buffer), writes `token` (default: this sampler's) and `history` if given."""
        if logits.device != self.device or logits.dtype != torch.float32 or logits.numel() < self.vocab:
            raise KernelError("logits must be float32 on the sampler's device with at least vocab entries")
        if not logits.is_contiguous():
            raise KernelError("logits must be contiguous")
        lib = library()
        stream = current_stream(self.device)
        check(lib.logit_bounds(stream, pointer(logits), pointer(self.temperature), pointer(self.penalty),
                               pointer(self.inverse_penalty), pointer(self.seen), pointer(self.bounds),
                               int32(self.vocab)), "logit_bounds")
        check(lib.sample_token(stream, pointer(logits), pointer(self.bounds), pointer(self.temperature),
                               pointer(self.penalty), pointer(self.inverse_penalty), pointer(self.seen),
                               pointer(self.top_k), pointer(self.uniform if uniform is None else uniform),
                               pointer(self.token if token is None else token), pointer(history),
                               int32(self.vocab)), "sample_token")

    def sample(self, logits: Tensor) -> int:
        """kernel_decoder.py:669-681: a fresh uniform, both launches, the token read back."""
        self.uniform.uniform_()
        self.launch(logits)
        return int(self.token[0])


class LogProbabilities(NamedTuple):
    """Of every row: log_probability and entropy [rows] (fp32, nats), and the likeliest tokens, falling:
    top_log_probability [rows, top] (fp32) and top_token [rows, top] (int64)."""

    log_probability: Tensor
    entropy: Tensor
    top_log_probability: Tensor
    top_token: Tensor


@functools.lru_cache(maxsize=4096)
def _score_workspace(*sizes: int) -> int:
    return library().ivonar_log_probabilities_work(*sizes)


def log_probabilities(logits: Tensor, tokens: Tensor, top: int = 0, temperature: float = 1.0) -> LogProbabilities:
    """Scores of tokens [rows] (int64) under softmax(logits / temperature), logits [rows, vocab] in fp32, fp16 or
    bfloat16 with any row stride.

    A token outside the vocabulary has the log probability -inf.  `top` (at most 64) alternatives are listed, of equal
    logits the lowest token first; a NaN counts as less than every number.  A row whose logits are all -inf has log
    probabilities of -inf and the entropy 0; a row with a NaN or +inf has NaN for all of its numbers, but for a token
    outside the vocabulary.  The fp32 results are parts of one tensor, which each of them keeps alive.  Nothing
    synchronises, and calls can be captured into a graph."""
    device = _device(logits, tokens)
    dtype = _DTYPES.get(logits.dtype)
    if logits.dim() != 2 or dtype is None or not 0 < logits.shape[1] <= 1 << 30:
        raise KernelError("logits must be float32, float16 or bfloat16 [rows, vocab]")
    rows, vocab = logits.shape
    if rows >= 1 << 31:
        raise KernelError("log_probabilities takes fewer than 2**31 rows")
    if logits.stride(1) != 1 and vocab > 1:
        raise KernelError("logits must have a row's values side by side")
    if tokens.dtype is not torch.int64 or tokens.shape != (rows,) or not tokens.is_contiguous():
        raise KernelError(f"tokens must be contiguous int64 [{rows}]")
    if not 0 <= top <= min(MAX_TOP, vocab):
        raise KernelError(f"top {top} outside 0..{min(MAX_TOP, vocab)}")
    if not (2e-38 < temperature < 1e38):
        raise KernelError("temperature must be positive and finite, and so must its inverse")
    numbers = tokens.new_empty((rows * (2 + top),), dtype=torch.float32)
    chosen, entropy, best = numbers.split_with_sizes((rows, rows, rows * top))
    best, token = best.view(rows, top), tokens.new_empty((rows, top))
    if rows:
        need = _score_workspace(dtype, rows, vocab, top)
        work = tokens.new_empty((need,), dtype=torch.uint8) if need > 0 else None
        _run("ivonar_log_probabilities", device, logits.data_ptr(), dtype, logits.stride(0), rows, vocab,
             tokens.data_ptr(), top, temperature, chosen.data_ptr(), entropy.data_ptr(), best.data_ptr(),
             token.data_ptr(), None if work is None else work.data_ptr(), need)
    return LogProbabilities(chosen, entropy, best, token)
