"""Alternatives of rows that begin with more logits that are no numbers than a wave looks at at a time."""

from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,vocab", [(4096, 5000), (2, 9000), (2, 32000), (1, 262144), (300, 9001)])
@pytest.mark.parametrize("behind", [2048, 4999, 8190])
def test_numbers_behind_others(cuda, dtype, rows, vocab, behind):
    """One wave for a row, several, sixteen, and several blocks; the numbers begin in a later chunk of any of them."""
    import torch
    from ivonar_amd import sampling

    if behind >= vocab:
        behind = vocab - 1
    few = min(rows, 3)
    logits = torch.full((few, vocab), float("nan"))
    logits[:, behind:] = torch.randn(few, vocab - behind, generator=torch.Generator().manual_seed(behind))
    logits[0, 2:5] = torch.tensor([0.5, -0.25, -float("inf")])  # numbers among the first, fewer than are asked for
    logits[-1, behind:] = logits[-1, behind:].abs().neg()
    logits = logits.to(getattr(torch, dtype)).to(cuda)
    all_rows = logits[torch.arange(rows, device=cuda) % few]
    tokens = torch.zeros(rows, dtype=torch.int64, device=cuda)
    order = torch.sort(torch.where(torch.isnan(logits.double()), -torch.inf, logits.double()), dim=1, descending=True,
                       stable=True).indices
    # -inf before what is no number, of those the lowest token first
    place = torch.arange(vocab, device=cuda)
    key = torch.where(torch.isnan(logits), 2, torch.where(logits == -torch.inf, 1, 0))
    expected = []
    for row in range(few):
        numbers = order[row][key[row][order[row]] == 0]
        expected.append(torch.cat((numbers, place[key[row] == 1], place[key[row] == 2])))
    expected = torch.stack(expected)
    for top in (1, 5, 20, 33, 64):
        got = sampling.log_probabilities(all_rows, tokens, top)
        assert torch.isnan(got.log_probability).all() and torch.isnan(got.top_log_probability).all()
        assert torch.equal(got.top_token, expected[torch.arange(rows, device=cuda) % few, :top]), f"top {top}"
