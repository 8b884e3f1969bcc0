"""Attention over shared prefixes against a plain 64-bit implementation that takes every sequence by itself."""

from __future__ import annotations

import numpy as np
import pytest

import _attention as A

pytestmark = pytest.mark.gpu

# Parts of a row are joined by factors of 2^(m1 - m), each right to 2^-22, which is four roundings: at most three in a
# block and one per part, of which there are up to 32 here.
JOINS = 4 * 40


def _ints(cuda, values):
    import torch

    return torch.tensor(values, dtype=torch.int32, device=cuda)


def _prefix(counts):
    return [0, *np.cumsum(counts).tolist()]


class Batch:
    """Sequences as (group, shared pages, tokens behind them, query rows); group None: outside all groups.  The groups'
    sequences are neighbours, in the order of their groups."""

    def __init__(self, cuda, rng, sequences, heads, kv, dim, page, dtype, groups=None, cut=None):
        import torch
        from ivonar_amd import attention

        self.cuda, self.dtype, self.kv = cuda, dtype, kv
        self.lengths = [shared * page + own for _, shared, own, _ in sequences]
        self.counts = [rows for *_, rows in sequences]
        count = (max((g for g, *_ in sequences if g is not None), default=-1) + 1) if groups is None else groups
        before, members = 0, [[b for b, s in enumerate(sequences) if s[0] == g] for g in range(count)]
        self.groups = []
        for of in members:
            before = of[0] if of else before
            self.groups.append(before)
            before = of[-1] + 1 if of else before
        self.groups.append(before)
        # the next group may begin further on: sequences between are in the one before, with nothing shared
        self.prefix = [sequences[of[0]][1] * page - (0 if cut is None else cut) if of else 77 for of in members]
        self.page, width = page, max(-(-n // page) for n in self.lengths) + 1
        pages, table = 0, np.full((len(sequences), width), -1, dtype=np.int32)
        order = rng.permutation(sum(-(-n // page) for n in self.lengths) + 3)
        first = {}
        for b, (group, shared, own, _) in enumerate(sequences):
            begin = 0
            if group is not None:
                if group in first:
                    table[b, :shared] = table[first[group], :shared]
                    begin = shared
                first.setdefault(group, b)
            needed = -(-self.lengths[b] // page)
            table[b, begin:needed] = order[pages:pages + needed - begin]
            pages += needed - begin
        self.pages = attention.cache_pages(len(order), kv, dim, page, cuda)
        self.pages.copy_(torch.randint(0, 256, self.pages.shape, dtype=torch.uint8))
        self.table = torch.from_numpy(table).to(cuda)
        self.k, self.v = [], []
        for b, (group, shared, own, _) in enumerate(sequences):
            k, v = (torch.randn(self.lengths[b], kv, dim) for _ in range(2))
            if group is not None and first[group] != b:
                for x, side in ((k, self.k), (v, self.v)):
                    x[:shared * page] = side[first[group]][:shared * page]
            self.k.append(k)
            self.v.append(v)
            self.write(b)
        self.q = torch.randn(sum(self.counts), heads, dim).to(getattr(torch, dtype)).to(cuda)

    def write(self, b):
        from ivonar_amd import attention

        attention.cache_write(self.pages, self.k[b].to(self.cuda), self.v[b].to(self.cuda), self.table[b:b + 1],
                              _ints(self.cuda, [0]), _ints(self.cuda, [0, self.lengths[b]]))

    def run(self, **options):
        from ivonar_amd import attention

        offsets = options.pop("offsets", _ints(self.cuda, _prefix(self.counts)))
        return attention.prefix_attention(options.pop("q", self.q), self.pages, self.table, _ints(self.cuda, self.lengths),
                                          _ints(self.cuda, options.pop("groups", self.groups)),
                                          _ints(self.cuda, options.pop("prefix", self.prefix)), offsets, **options)

    def check(self, out, what="", some=None, scale=None, missing=None):
        rows = _prefix(self.counts)
        q = self.q.double().cpu().numpy()
        for b in range(len(self.counts)) if some is None else some:
            if not self.counts[b]:
                continue
            k, v = (A.stored(x[b].numpy()) for x in (self.k, self.v))
            part = slice(rows[b], rows[b + 1])
            expected = A.attend(q[part], k, v, self.lengths[b] - self.counts[b], scale=scale,
                                missing=None if missing is None else missing[b])
            A.check(out[part].double().cpu().numpy(), *expected, self.dtype, self.lengths[b] + JOINS, q.shape[2],
                    f"{what} sequence {b}")


TWO_GROUPS = [(None, 0, 40, 1), (0, 2, 5, 1), (0, 2, 70, 1), (0, 2, 1, 1), (None, 0, 1, 1), (1, 3, 33, 1), (1, 3, 32, 1),
              (None, 0, 100, 1)]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("dim,heads,kv,page", [(64, 4, 4, 32), (64, 14, 2, 64), (128, 8, 2, 32), (128, 3, 1, 128),
                                               (256, 4, 2, 32), (256, 20, 1, 64)])
def test_groups_and_others(cuda, rng, dtype, dim, heads, kv, page):
    """Two groups with sequences outside them before, between and behind; one row each, and a few."""
    for rows in (1, 4):
        sequences = [(g, shared, max(own, rows), rows) for g, shared, own, _ in TWO_GROUPS]
        batch = Batch(cuda, rng, sequences, heads, kv, dim, page, dtype)
        batch.groups, batch.prefix = [1, 4, 5, 7], [2 * page, 0, 3 * page]
        batch.check(batch.run(), f"{rows} rows")
        if rows == 1:
            batch.check(batch.run(offsets=None), "no offsets")


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("dim,heads,kv", [(64, 16, 16), (128, 8, 2), (256, 8, 2)])
def test_many_rows_of_a_group(cuda, rng, dtype, dim, heads, kv):
    """Row tiles that hold several sequences' rows, and prefixes split between blocks."""
    sequences = [(0, 40, 1 + 7 * b % 50, 1) for b in range(21)]
    batch = Batch(cuda, rng, sequences, heads, kv, dim, 32, dtype)
    batch.check(batch.run(max_prefix=1280, max_length=1330), "21 sequences")
    batch.check(batch.run(), "no hints", some=[0, 7, 20])


@pytest.mark.parametrize("cut", [1, 31, 32, 40, 63, 64, 127])
def test_prefix_ends_anywhere(cuda, rng, cut):
    """Fewer tokens than the pages share, within tiles and pages, and none."""
    batch = Batch(cuda, rng, [(0, 2, 3 + 40 * b, 1) for b in range(5)], 4, 2, 64, 64, "float32", cut=cut)
    batch.check(batch.run(), f"cut {cut}")
    batch.check(batch.run(prefix=[0]), "nothing shared")
    batch.check(batch.run(prefix=[-5]), "less than nothing")


def test_rows_within_the_prefix(cuda, rng):
    """Rows that begin before the prefix ends see what lies before them, and so do the others of their group."""
    sequences = [(0, 3, 0, 20), (0, 3, 2, 5), (0, 3, 40, 2), (1, 2, 0, 64), (1, 2, 9, 1)]
    for dtype in ("float32", "bfloat16"):
        batch = Batch(cuda, rng, sequences, 4, 2, 64, 32, dtype)
        batch.check(batch.run(), dtype)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_sequences_without_rows_and_tokens(cuda, rng, dtype):
    """Groups none of whose sequences have rows, empty groups, sequences of no tokens, and padding behind the last."""
    import torch

    sequences = [(0, 2, 5, 0), (0, 2, 9, 0), (1, 1, 1, 1), (1, 1, 30, 0), (1, 1, 7, 2), (None, 0, 3, 3)]
    batch = Batch(cuda, rng, sequences, 4, 1, 128, 32, dtype)
    batch.groups, batch.prefix = [0, 2, 2, 2, 5], [64, 10, 10, 32]
    batch.check(batch.run())
    padded = torch.cat((batch.q, batch.q[:3] * float("nan")))
    out = batch.run(q=padded)
    assert not out[len(batch.q):].any()
    batch.check(out[:len(batch.q)])
    lengths, batch.lengths = batch.lengths, [0] * 6
    assert not batch.run().any()
    batch.lengths = lengths
    none = batch.run(q=batch.q[:0], offsets=_ints(cuda, [0] * 7))
    assert none.shape == (0, 4, 128)
    batch.check(batch.run(groups=[0], prefix=[]), "no groups")
    batch.check(batch.run(groups=[6], prefix=[]), "no groups")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("dead", [[0], [1, 3], [0, 1, 2, 3], [0, 2, 4, 5]])
def test_padded_batch(cuda, rng, dtype, dead):
    """Sequences of no tokens and no pages but with a row each, as a batch of a fixed size has: first in a group, in the
    middle, and whole groups of them."""
    sequences = [(0, 4, 5 + 9 * b, 1) for b in range(4)] + [(1, 2, 40, 1), (1, 2, 3, 1)]
    batch = Batch(cuda, rng, sequences, 8, 2, 64, 32, dtype)
    for b in dead:
        batch.lengths[b] = 0
        batch.table[b] = -1
    live = [b for b in range(6) if b not in dead]
    for offsets in (None, _ints(cuda, list(range(7)))):
        for hints in ({}, {"max_prefix": 128, "max_length": 200}):
            out = batch.run(offsets=offsets, **hints)
            assert not out[dead].any()
            batch.check(out, some=live)


def test_many_groups(cuda, rng):
    """More groups and sequences than a wave has lanes, of one to three sequences."""
    sequences, b = [], 0
    for group in range(150):
        for _ in range(1 + group % 3):
            sequences.append((group, group % 4, 1 + (b * 13) % 60, 1))
            b += 1
    batch = Batch(cuda, rng, sequences, 2, 1, 64, 32, "bfloat16")
    out = batch.run()
    batch.check(out, some=[*range(0, len(sequences), 7), len(sequences) - 1])
    batch.check(batch.run(offsets=None), some=[0, 5, 100, len(sequences) - 1])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 64), (8, 2, 128), (2, 1, 256)])
def test_long_tails(cuda, rng, dtype, heads, kv, dim):
    """Tails that are split between blocks, of one row and of several row tiles, behind a short prefix."""
    for rows in (1, 40):
        batch = Batch(cuda, rng, [(0, 1, 1500, rows), (0, 1, 47, rows), (None, 0, 900, rows)], heads, kv, dim, 32, dtype)
        batch.check(batch.run(max_prefix=32), f"{rows} rows")
        batch.check(batch.run(max_prefix=0, max_length=1), "hints of nothing")


def test_hints_do_not_matter(cuda, rng):
    batch = Batch(cuda, rng, [(0, 20, 3 + b, 1) for b in range(9)], 8, 2, 64, 32, "float32")
    for hints in ((0, 1), (1, 10 ** 9), (640, 650), (10 ** 9, 10 ** 9), (100, 200)):
        batch.check(batch.run(max_prefix=hints[0], max_length=hints[1]), str(hints), some=[0, 8])


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_missing_pages_and_not_numbers(cuda, rng, dtype):
    """Entries without a page in the prefix and behind it are not seen; a NaN reaches the rows that see it and no other."""
    batch = Batch(cuda, rng, [(0, 4, 50, 1), (0, 4, 20, 1), (1, 4, 40, 2), (1, 4, 41, 1)], 4, 2, 64, 32, dtype)
    missing = [np.zeros(n, dtype=bool) for n in batch.lengths]
    batch.table[:2, 1] = -1
    batch.table[0, 4] = 1 << 20
    for b, begin, end in ((0, 32, 64), (1, 32, 64), (0, 128, 160)):
        missing[b][begin:end] = True
    batch.check(batch.run(), "missing", missing=missing)
    whole = batch.run()
    for place, seen_by in ((100, [2, 3, 4]), (150, [2, 3])):  # in the second group's prefix, and behind it in its first
        for side in (batch.k, batch.v):
            kept = side[2][place, 0, 3].clone()
            side[2][place, 0, 3] = float("nan")
            batch.write(2)
            out = batch.run()
            side[2][place, 0, 3] = kept
            batch.write(2)
            odd = ~np.isfinite(out.float().cpu().numpy()).all(-1)
            expected = np.zeros_like(odd)
            expected[seen_by, :2] = True  # the heads that share the first key/value head
            assert np.array_equal(odd, expected), (place, np.argwhere(odd != expected))
            kept_rows = [r for r in range(5) if r not in seen_by]
            assert np.array_equal(out[kept_rows].float().cpu().numpy(), whole[kept_rows].float().cpu().numpy())


def test_against_cache_attention(cuda, rng):
    """Strided queries, a scale, a given output; within both calls' bounds of each other."""
    import torch
    from ivonar_amd import attention

    batch = Batch(cuda, rng, [(0, 6, 5 + 9 * b, 2) for b in range(7)], 8, 2, 128, 64, "bfloat16")
    fused = torch.randn(14, 24, 128, device=cuda).bfloat16()
    fused[:, 3:11] = batch.q
    at = (batch.pages, batch.table, _ints(cuda, batch.lengths))
    offsets = _ints(cuda, _prefix(batch.counts))
    out = torch.empty_like(batch.q)
    assert batch.run(q=fused[:, 3:11], scale=0.3, out=out) is out
    batch.check(out, scale=0.3)
    other = attention.cache_attention(batch.q, *at, offsets, scale=0.3)
    assert (out.float() - other.float()).abs().max() < 0.05
    odd = torch.cat([fused.flatten(), fused.new_zeros(1)])[1:].view(fused.shape)
    odd[:, 3:11] = batch.q
    assert torch.equal(batch.run(q=odd[:, 3:11], scale=0.3), out)


def test_infinite_logits_and_large_ones(cuda, rng):
    """Logits whose maximum fp32 rounds by whole numbers, in the prefix and behind it."""
    import torch
    from ivonar_amd import attention

    pages = attention.cache_pages(4, 1, 64, 32, cuda)
    table = _ints(cuda, [[0, 1, 2], [0, 1, 3]])
    k = torch.zeros(70, 1, 64, device=cuda)
    k[:, 0, 0] = 1
    k[10, 0, 1], k[66, 0, 1] = 1, 1
    v = torch.arange(70, device=cuda).float().view(-1, 1, 1).expand(70, 1, 64).contiguous()
    for row in range(2):
        attention.cache_write(pages, k, v, table[row:row + 1], _ints(cuda, [0]), _ints(cuda, [0, 70]))
    q = torch.zeros(2, 1, 64, device=cuda)
    q[:, 0, 0], q[:, 0, 1] = 2.0 ** 30, 2.0 ** 8
    out = attention.prefix_attention(q, pages, table, _ints(cuda, [70, 66]), _ints(cuda, [0, 2]), _ints(cuda, [64]),
                                     scale=1.0)
    kept = A.stored(v.cpu().numpy())
    assert torch.allclose(out[0].cpu().double(), torch.from_numpy((kept[10] + kept[66]) / 2), rtol=1e-6)
    assert torch.equal(out[1].cpu().double(), torch.from_numpy(kept[10]))


def test_streams_and_graphs(cuda, rng):
    """Two calls at once on two streams, and a captured one replayed with other rows, lengths and prefixes in place."""
    import torch
    from ivonar_amd import attention

    batches = [Batch(cuda, rng, [(0, 10, 5 + b, 1) for b in range(n)], 8, 2, 64, 32, "bfloat16") for n in (6, 30)]
    at = [(b.q, b.pages, b.table, _ints(cuda, b.lengths), _ints(cuda, b.groups), _ints(cuda, b.prefix)) for b in batches]
    expected = [attention.prefix_attention(*a) for a in at]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for _ in range(5):
        for stream, a in zip(streams, at):
            with torch.cuda.stream(stream):
                results.append(attention.prefix_attention(*a))
    torch.cuda.synchronize()
    for i, got in enumerate(results):
        assert torch.equal(got, expected[i % 2])
    batch = batches[0]
    q, lengths, prefix = batch.q.clone(), _ints(cuda, batch.lengths), _ints(cuda, batch.prefix)
    groups = _ints(cuda, batch.groups)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attention.prefix_attention(q, batch.pages, batch.table, lengths, groups, prefix)
    full = list(batch.lengths)
    for replay in range(4):
        batch.q = torch.randn_like(q, dtype=torch.float32).bfloat16()
        batch.lengths = [n - replay for n in full]
        kept = batch.k, batch.v
        batch.k, batch.v = ([x[:n] for x, n in zip(side, batch.lengths)] for side in kept)
        q.copy_(batch.q)
        lengths.copy_(_ints(cuda, batch.lengths))
        prefix.fill_(320 - 50 * replay)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        batch.check(out, f"replay {replay}")
        batch.k, batch.v = kept


def test_refusals(cuda, rng):
    import torch
    from ivonar_amd import attention
    from ivonar_amd.runtime import KernelError

    batch = Batch(cuda, rng, [(0, 1, 3, 2), (0, 1, 4, 2)], 4, 2, 64, 32, "float32")
    good = dict(q=batch.q, pages=batch.pages, table=batch.table, lengths=_ints(cuda, batch.lengths),
                groups=_ints(cuda, [0, 2]), prefix=_ints(cuda, [32]), offsets=_ints(cuda, [0, 2, 4]))
    attention.prefix_attention(**good)
    for name, value in (("q", batch.q[..., :32]), ("q", batch.q[:, :3]), ("q", batch.q.double()), ("q", batch.q.cpu()),
                        ("q", batch.q[:, :0]), ("pages", batch.pages.float()), ("pages", batch.pages[..., :-2]),
                        ("table", batch.table.long()), ("lengths", good["lengths"][:1]), ("offsets", None),
                        ("offsets", good["offsets"][:2]), ("groups", _ints(cuda, [0])), ("groups", _ints(cuda, [0, 1, 2])),
                        ("groups", good["groups"].long()), ("prefix", good["prefix"].long()),
                        ("prefix", _ints(cuda, [32, 32])), ("prefix", good["prefix"][0]), ("prefix", good["prefix"].cpu()),
                        ("scale", 0.0), ("scale", float("nan")), ("out", batch.q[:3]), ("out", batch.q.half())):
        with pytest.raises(KernelError):
            attention.prefix_attention(**{**good, name: value})
    with pytest.raises(KernelError):  # more groups than sequences
        attention.prefix_attention(**{**good, "groups": _ints(cuda, [0, 1, 2, 2]), "prefix": _ints(cuda, [0, 0, 0])})
    bad = torch.empty(batch.q.numel() + 1, device=cuda)[1:].view(batch.q.shape)
    with pytest.raises(KernelError):
        attention.prefix_attention(**good, out=bad)
