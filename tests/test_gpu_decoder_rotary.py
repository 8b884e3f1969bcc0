"""The decoder with rotated queries and keys, and its scores of a prompt's tokens."""

from __future__ import annotations

import numpy as np
import pytest

import _attention as A
from ivonar_amd.synthetic import StackConfig, decoder_stack, prompt_ids

pytestmark = pytest.mark.gpu

STACK = StackConfig(vocab=700, hidden=256, layers=2, dense=512)


def _decoder(cuda, attention=True, burst=8, **options):
    from ivonar_amd.decoder import AttentionConfig, StackDecoder

    config = AttentionConfig(4, **{"rotary_base": 10000.0, **options}) if attention else None
    return StackDecoder(decoder_stack(STACK, seed=3), cuda, burst=burst, attention=config)


class Watch:
    """Checks every attention call of a decoder that runs eagerly, from the projections' rows that it was given, rotated
    by rotate() apart."""

    def __init__(self, decoder) -> None:
        self.attention = attention = decoder.attention
        self.rows = [[] for _ in decoder.layers]
        self.calls = 0
        step, tile = attention.step, attention.tile

        def watched_step(layer, mixer_in):
            new = self.rotated(mixer_in.unsqueeze(0).clone(), int(attention.step_index[0]))
            step(layer, mixer_in)
            self.check(layer, new, attention.mixed.unsqueeze(0), int(attention.step_index[0]))

        def watched_tile(layer, mixer_in, first):
            start, _, _, count = attention.tile_index.tolist()
            new = self.rotated(mixer_in[:count].clone(), start)
            tile(layer, mixer_in, first)
            if start == 0:
                self.rows[layer] = []
            self.check(layer, new, attention.mixed_tile[:count], start, first)

        attention.step, attention.tile = watched_step, watched_tile

    def rotated(self, rows, start):
        import torch
        from ivonar_amd import attention

        q, k, v = rows.unflatten(1, (3, *self.attention.shape)).unbind(1)
        index = torch.tensor([start, 0, rows.shape[0]], dtype=torch.int32, device=rows.device)
        frequencies = attention.rotary_frequencies(self.attention.shape[1], self.attention.config.rotary_base,
                                                   device=rows.device)
        return torch.stack((*attention.rotate(q, k, index[:1], frequencies, index[1:]), v), 1)

    def check(self, layer, new, mixed, start, first=False):
        config, shape = self.attention.config, self.attention.shape
        rows = new.cpu().numpy()
        kept = self.rows[layer][:start]
        assert len(kept) == start
        self.rows[layer] = kept + list(rows)
        history = np.stack(self.rows[layer])
        if first:
            q, k, v = new.bfloat16().float().cpu().numpy().transpose(1, 0, 2, 3)
        else:
            q, k, v = rows[:, 0], A.stored(history[:, 1]), A.stored(history[:, 2])
        result = A.attend(q, k, v, start, config.window, config.sinks)
        dtype, more = ("bfloat16", {"weight_unit": 2.0 ** -8}) if first else ("float32", {})
        A.check(mixed.cpu().numpy().reshape(-1, *shape), *result, dtype, len(history), shape[1], f"layer {layer}", **more)
        self.calls += 1


@pytest.mark.parametrize("options", [{}, {"window": 20, "sinks": 3, "page_size": 32, "rotary_base": 500.0}])
def test_every_call(cuda, monkeypatch, options):
    """A prompt in three tiles, then steps."""
    from ivonar_amd import decoder as module

    monkeypatch.setattr(module, "TILES", (32, 64))
    decoder = _decoder(cuda, **options)
    watch = Watch(decoder)
    layers = decoder._build_layers()
    decoder._steps = [decoder._build_step(slot, layers) for slot in range(decoder.burst)]
    decoder._tiles, decoder._later_tiles = decoder._build_tiles(), decoder._build_tiles(first=False)
    tokens = decoder.generate(prompt_ids(STACK.vocab, 141, seed=2), 10)
    assert watch.calls == STACK.layers * (3 + 9)
    assert all(0 <= token < STACK.vocab for token in tokens)


def test_graphs_match_eager_runs(cuda):
    import torch

    prompts = [prompt_ids(STACK.vocab, n, seed=n) for n in (36, 1100, 5)]
    decoder = _decoder(cuda)
    eager = [decoder.generate(prompt, 20) for prompt in prompts]
    scores = [decoder.score(prompt, 3) for prompt in prompts]
    decoder.prefill(prompts[0])
    decoder.capture()
    first = [int(decoder.history[decoder.burst - 1])]
    assert first + decoder.advance_many(19) == eager[0]
    for turn in range(2):
        for prompt, tokens, score in zip(prompts, eager, scores):
            assert decoder.generate(prompt, 20) == tokens, turn
            for a, b in zip(decoder.score(prompt, 3), score):
                assert torch.equal(a, b), turn
            assert decoder.advance_many(19) == tokens[1:]
    decoder.self_check()


def test_rotation_changes_the_tokens(cuda):
    """Positions count: with and without them the same prompt ends in other logits."""
    import torch

    prompt = prompt_ids(STACK.vocab, 50)
    turned, plain = (_decoder(cuda, rotary_base=base).prefill(prompt).clone() for base in (10000.0, 0.0))
    assert not torch.equal(turned, plain)


@pytest.mark.parametrize("attention", [False, True])
def test_scores_are_those_of_the_logits(cuda, monkeypatch, attention):
    """At the ends of tiles, where a shorter prompt runs in the same tiles and its last logits come from the decode
    head: the same int8 products, summed in fp32 in another order (two groups of 128 inputs: four roundings of the
    terms' size, which is within 2^-20 of the largest logit's)."""
    import torch
    from ivonar_amd import decoder as module

    monkeypatch.setattr(module, "TILES", (32, 64))
    decoder = _decoder(cuda, attention)
    ids = prompt_ids(STACK.vocab, 142, seed=4)
    got = decoder.score(ids, 5)
    assert got.log_probability.shape == got.entropy.shape == (141,)
    assert got.top_log_probability.shape == got.top_token.shape == (141, 5)
    tokens = decoder.advance_many(5)
    for n in (64, 128, 141):
        prefix = ids[:n]
        logits = decoder.prefill(prefix).double()
        logs = torch.log_softmax(logits, 0)
        limit = 2.0 ** -18 * float(logits.abs().max()) + 2.0 ** -18
        assert abs(float(got.log_probability[n - 1]) - float(logs[int(ids[n])])) <= limit, n
        best = torch.sort(logs, descending=True, stable=True)
        assert (got.top_log_probability[n - 1].double() - best.values[:5]).abs().max() <= limit
        assert abs(float(got.entropy[n - 1]) + float((logs.exp() * logs).sum())) <= 16 * limit
    decoder.prefill(ids)
    assert decoder.advance_many(5) == tokens  # score leaves the decoder as prefill does


def test_score_refusals_and_short_prompts(cuda):
    from ivonar_amd.runtime import KernelError

    decoder = _decoder(cuda, capacity=40)
    one = decoder.score([5], 3)
    assert one.log_probability.shape == (0,) and one.top_token.shape == (0, 3)
    assert decoder.score([5, 6]).log_probability.shape == (1,)
    for top in (-1, 65):
        with pytest.raises(KernelError):
            decoder.score([5, 6], top)
    for bad, error in (([], ValueError), ([700], IndexError), ([1] * 41, ValueError)):
        with pytest.raises(error):
            decoder.score(bad)
    for base in (-1.0, float("nan"), float("inf")):
        with pytest.raises(KernelError):
            _decoder(cuda, rotary_base=base)
