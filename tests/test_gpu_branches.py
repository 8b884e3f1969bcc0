"""One prompt that goes on in many ways: rotated keys and queries into the cache, pages reserved and forked, attention
over the shared prefix, logits scored, branches pruned, pages moved together; step by step against 64-bit attention."""

from __future__ import annotations

import numpy as np
import pytest

import _attention as A
from test_gpu_score import check as check_scores

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, PAGE, VOCAB = 8, 2, 64, 32, 1500
JOINS = 4 * 40


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_prompt_goes_on_in_many_ways(cuda, dtype):
    import torch
    from ivonar_amd import attention, paging, sampling
    from ivonar_amd.quantization import TernaryLinear, pack_ternary_codes

    kind = getattr(torch, dtype)
    generator = torch.Generator().manual_seed(7)
    weight = (torch.rand(VOCAB, HEADS * DIM, generator=generator) * 3).long() - 1
    head = TernaryLinear(pack_ternary_codes(weight), torch.full((VOCAB, HEADS * DIM // 128), 0.05).half(),
                         HEADS * DIM).to(cuda)
    norms = [(1 + 0.2 * torch.randn(DIM, generator=generator)).to(cuda) for _ in range(2)]
    frequencies = attention.rotary_frequencies(DIM, device=cuda)
    layers = [attention.cache_pages(60, KV, DIM, PAGE, cuda) for _ in range(2)]
    pool = paging.page_pool(60, PAGE, cuda)
    table = torch.full((1, 12), -1, dtype=torch.int32, device=cuda)
    lengths = torch.zeros(1, dtype=torch.int32, device=cuda)
    history = [[(np.zeros((0, KV, DIM)), np.zeros((0, KV, DIM))) for _ in layers]]  # of each sequence: keys, values

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=cuda)

    def new_tokens(counts, shared):
        """counts[b] new tokens of each sequence through all layers; their last layer's attention."""
        nonlocal lengths, table
        rows = sum(counts)
        offsets = ints([0, *np.cumsum(counts).tolist()])
        assert int(paging.reserve(pool, table, lengths, ints(counts))) == 0
        after = lengths + ints(counts)
        for layer, pages in enumerate(layers):
            q, k, v = (torch.randn(rows, n, DIM, generator=generator).to(kind).to(cuda) for n in (HEADS, KV, KV))
            turned_q, turned_k = attention.rotate(q, k, lengths, frequencies, offsets, *norms)
            written = attention.rotate_write(pages, q, k, v, table, lengths, frequencies, offsets, *norms)
            assert torch.equal(written, turned_q)
            keys, values = A.stored(turned_k.float().cpu().numpy()), A.stored(v.float().cpu().numpy())
            out = attention.prefix_attention(written, pages, table, after, ints([0, len(counts)]), ints([shared]), offsets)
            begin = 0
            for b, count in enumerate(counts):
                part = slice(begin, begin + count)
                begin += count
                old = history[b][layer]
                history[b][layer] = tuple(np.concatenate((x, y[part])) for x, y in zip(old, (keys, values)))
                if count > 0:
                    last = slice(part.stop - min(count, 3), part.stop)
                    rows_q = written[last].double().cpu().numpy()
                    first = len(history[b][layer][0]) - rows_q.shape[0]
                    expected = A.attend(rows_q, *history[b][layer], first)
                    A.check(out[last].double().cpu().numpy(), *expected, dtype, first + JOINS, DIM, f"{layer} {b}")
        lengths = after
        return out

    def go_on(parents):
        nonlocal lengths, table, history
        before = [len(h[0][0]) for h in history]
        table, lengths, copies, missing = paging.fork(pool, table, lengths, ints(parents))
        assert int(missing) == 0
        for pages in layers:
            paging.copy(pages, copies)
        history = [[tuple(x.copy() for x in layer) for layer in history[p]] for p in parents]
        assert lengths.tolist() == [before[p] for p in parents]

    new_tokens([83], 0)
    go_on([0] * 6)
    shared = 83 // PAGE * PAGE
    for step in range(9):
        out = new_tokens([1 + step % 2] * len(history), shared)
        logits = head(out.flatten(1).float())
        tokens = torch.randint(0, VOCAB, (logits.shape[0],), generator=generator).to(cuda)
        check_scores(sampling.log_probabilities(logits, tokens, 4, 0.9), logits, tokens, 4, 0.9, f"step {step}")
        if step == 3:  # the better branches twice, the others no more
            go_on([0, 0, 2, 2, 5])
        if step == 5:
            copies, held = paging.compact(pool, table)
            for pages in layers:
                paging.copy(pages, copies)
            assert int(held) == int((pool.refs > 0).sum()) and not pool.refs[int(held):].any()
    paging.release(pool, table)
    assert not pool.refs.any()


def test_cache_past_32_bits(cuda):
    """Pages that lie 4 GiB and more into the cache: rotated keys written there, and read as a shared prefix."""
    import torch
    from ivonar_amd import attention

    generator = torch.Generator().manual_seed(3)
    pages = torch.empty((2200, 16, 4, 34 * 256), dtype=torch.uint8, device=cuda)  # 1.2 GB
    pages = torch.cat((pages, pages, pages, pages))  # 4.9 GB, 557056 bytes a page
    count = pages.shape[0]
    assert pages.numel() > 1 << 32
    last = [count - 1, count - 7, 5, count - 2]  # shared, shared, and of either sequence
    table = torch.tensor([last[:2] + [last[2]], last[:2] + [last[3]]], dtype=torch.int32, device=cuda)
    frequencies = attention.rotary_frequencies(256, device=cuda)

    def ints(*values):
        return torch.tensor(values, dtype=torch.int32, device=cuda)

    q, k, v = (torch.randn(300, n, 256, generator=generator).to(cuda) for n in (16, 16, 16))
    offsets = ints(0, 290, 290)
    _, turned = attention.rotate(q[:290], k[:290], ints(0, 256), frequencies, offsets)
    attention.rotate_write(pages, q[:290], k[:290], v[:290], table, ints(0, 256), frequencies, offsets)
    _, more = attention.rotate(q[290:], k[290:], ints(256, 256), frequencies, ints(0, 0, 10))
    attention.rotate_write(pages, q[290:], k[290:], v[290:], table, ints(256, 256), frequencies, ints(0, 0, 10))
    rows = torch.randn(2, 16, 256, generator=generator).to(cuda)
    out = attention.prefix_attention(rows, pages, table, ints(290, 266), ints(0, 2), ints(256))
    for b, (own, value) in enumerate(((turned, v[:290]), (torch.cat((turned[:256], more)), torch.cat((v[:256], v[290:]))))):
        keys, values = A.stored(own.cpu().numpy()), A.stored(value.cpu().numpy())
        expected = A.attend(rows[b:b + 1].double().cpu().numpy(), keys, values, len(keys) - 1)
        A.check(out[b:b + 1].double().cpu().numpy(), *expected, "float32", len(keys) + JOINS, 256, f"sequence {b}")
