"""The decoder with attention between its linears: every attention result against 64-bit attention over the keys and
values that the decoder produced, and graphs against eager runs."""

from __future__ import annotations

import numpy as np
import pytest

import _attention as A
from ivonar_amd.synthetic import StackConfig, decoder_stack, prompt_ids

pytestmark = pytest.mark.gpu

STACK = StackConfig(vocab=700, hidden=256, layers=2, dense=512)


def _decoder(cuda, heads=4, burst=8, sampling=False, **options):
    from ivonar_amd.decoder import AttentionConfig, StackDecoder

    return StackDecoder(decoder_stack(STACK, seed=3), cuda, burst=burst, sampling=sampling,
                        attention=AttentionConfig(heads, **options))


class Watch:
    """Checks every attention call of a decoder that runs eagerly, from the projections' rows that it was given."""

    def __init__(self, decoder) -> None:
        self.attention = attention = decoder.attention
        self.rows = [[] for _ in decoder.layers]
        self.calls = 0
        step, tile = attention.step, attention.tile

        def watched_step(layer, mixer_in):
            step(layer, mixer_in)
            self.check(layer, mixer_in.unsqueeze(0), attention.mixed.unsqueeze(0), int(attention.step_index[0]))

        def watched_tile(layer, mixer_in, first):
            tile(layer, mixer_in, first)
            start, _, _, count = attention.tile_index.tolist()
            if start == 0:
                self.rows[layer] = []
            self.check(layer, mixer_in[:count], attention.mixed_tile[:count], start, first)
            assert not attention.mixed_tile[count:mixer_in.shape[0]].any()

        attention.step, attention.tile = watched_step, watched_tile

    def check(self, layer, mixer_in, mixed, start, first=False):
        config, shape = self.attention.config, self.attention.shape
        new = mixer_in.float().cpu().numpy().reshape(-1, 3, *shape)
        kept = self.rows[layer][:start]
        assert len(kept) == start
        self.rows[layer] = kept + list(new)
        history = np.stack(self.rows[layer])
        if first:  # the prompt's own rows in bfloat16
            history = mixer_in.bfloat16().float().cpu().numpy().reshape(-1, 3, *shape)
            q, k, v = history[:, 0], history[:, 1], history[:, 2]
        else:
            q, k, v = new[:, 0], A.stored(history[:, 1]), A.stored(history[:, 2])
        result = A.attend(q, k, v, start, config.window, config.sinks)
        dtype, more = ("bfloat16", {"weight_unit": 2.0 ** -8}) if first else ("float32", {})
        A.check(mixed.cpu().numpy().reshape(-1, *shape), *result, dtype, len(history), shape[1], f"layer {layer}", **more)
        self.calls += 1


@pytest.mark.parametrize("options", [{}, {"window": 20, "sinks": 3, "page_size": 32}, {"heads": 2, "capacity": 200}])
def test_every_call(cuda, monkeypatch, options):
    """A prompt in three tiles, then steps."""
    from ivonar_amd import decoder as module

    monkeypatch.setattr(module, "TILES", (32, 64))
    decoder = _decoder(cuda, **options)
    # the launch lists hold the methods themselves: watch, then build them again
    watch = Watch(decoder)
    layers = decoder._build_layers()
    decoder._steps = [decoder._build_step(slot, layers) for slot in range(decoder.burst)]
    decoder._tiles, decoder._later_tiles = decoder._build_tiles(), decoder._build_tiles(first=False)
    tokens = decoder.generate(prompt_ids(STACK.vocab, 141, seed=2), 10)
    assert watch.calls == STACK.layers * (3 + 9)
    assert decoder.attention.tokens == 141 + 9
    assert all(0 <= token < STACK.vocab for token in tokens)


@pytest.mark.parametrize("sampling", [False, True])
def test_graphs_match_eager_runs(cuda, sampling):
    import torch

    prompts = [prompt_ids(STACK.vocab, n, seed=n) for n in (36, 1100, 5)]
    decoder = _decoder(cuda, sampling=sampling, window=64, sinks=4)
    if sampling:
        decoder.configure_sampling(0.7, 1)  # the most likely token, drawn
    eager = [decoder.generate(prompt, 20) for prompt in prompts]
    decoder.prefill(prompts[0])
    decoder.capture()
    assert decoder.attention.tokens == 36
    first = [int(decoder.history[decoder.burst - 1])]
    assert first + decoder.advance_many(19) == eager[0]  # the cache outlives the capture
    for turn in range(2):
        for prompt, tokens in zip(prompts, eager):
            assert decoder.generate(prompt, 20) == tokens, turn
            torch.cuda.synchronize()


def test_self_check_and_reset(cuda):
    decoder = _decoder(cuda)
    decoder.self_check()
    assert decoder.attention.tokens == 0
    decoder.history.fill_(7)
    decoder.step()
    assert decoder.attention.tokens == 1
    assert decoder.attention.step_index.tolist() == [1, 2]


def test_refusals(cuda):
    from ivonar_amd.runtime import KernelError

    for options in ({"heads": 3}, {"heads": 0}, {"heads": 8}, {"heads": 4, "capacity": 0}, {"heads": 4, "page_size": 40}):
        with pytest.raises(KernelError):
            _decoder(cuda, **options)
    decoder = _decoder(cuda, capacity=40)
    with pytest.raises(ValueError):
        decoder.prefill(prompt_ids(STACK.vocab, 41))
    decoder.generate(prompt_ids(STACK.vocab, 38), 3)
    with pytest.raises(ValueError):
        decoder.step()
    assert decoder.attention.tokens == 40
    decoder.prefill(prompt_ids(STACK.vocab, 40))  # a new prompt starts anew


def test_refused_prompt_leaves_the_sequence_as_it_is(cuda):
    decoder = _decoder(cuda, capacity=40)
    decoder.generate(prompt_ids(STACK.vocab, 36), 3)
    with pytest.raises(ValueError):
        decoder.prefill(prompt_ids(STACK.vocab, 41))
    assert decoder.attention.tokens == 38 == int(decoder.attention.step_index[0])
    decoder.step()
    decoder.step()
    with pytest.raises(ValueError):
        decoder.step()
    assert decoder.attention.tokens == 40 == int(decoder.attention.step_index[0])


@pytest.mark.parametrize("captured", [False, True])
def test_many_steps_are_refused_as_a_whole(cuda, captured):
    """No token is lost where the cache has room for some of a call's steps only."""
    prompt = prompt_ids(STACK.vocab, 20)
    expected = _decoder(cuda).generate(prompt, 21)
    decoder = _decoder(cuda, capacity=40)
    decoder.prefill(prompt)
    if captured:
        decoder.capture()
    first = int(decoder.history[decoder.burst - 1])
    with pytest.raises(ValueError):
        decoder.advance_many(21)
    assert decoder.attention.tokens == 20 == int(decoder.attention.step_index[0])
    assert [first] + decoder.advance_many(20) == expected
    with pytest.raises(ValueError):
        decoder.advance_many(1)
    with pytest.raises(ValueError):
        decoder.generate(prompt, 22)
    assert decoder.generate(prompt, 21) == expected


@pytest.mark.parametrize("capacity", [1, 2, 33, 48])
def test_self_check_of_a_small_cache(cuda, capacity):
    decoder = _decoder(cuda, capacity=capacity)
    decoder.self_check()
    assert decoder.attention.tokens == 0


@pytest.mark.parametrize("layers,dense,seed", [(16, 256, 17), (6, 512, 2)])
def test_self_check_allows_for_the_cache(cuda, layers, dense, seed):
    """Stacks whose steps, with keys and values in 4 bits, are further from the prompt's tile than without a cache."""
    from ivonar_amd.decoder import AttentionConfig, StackDecoder

    weights = decoder_stack(StackConfig(vocab=700, hidden=64, layers=layers, dense=dense), seed=seed)
    StackDecoder(weights, cuda, attention=AttentionConfig(1)).self_check()
