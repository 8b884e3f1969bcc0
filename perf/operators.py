"""The attention operators of a decoder and its 4-bit cache, as cases to be measured.

Four kinds of case, each through the package's public entry points:

* ``write``: the keys and values of new tokens quantised into the cache's pages, and read back as attention will
  see them (the round trip that a program makes when it keeps a prompt's cache for later);
* ``read``: stretches of cached sequences read back as ordinary tensors;
* ``cache``: attention of a few query tokens of each sequence over its cached tokens, all of them or a sliding
  window and the first few (sinks);
* ``prompt``: attention within packed prompts over their unquantised keys and values, causal, with or without a
  window and sinks.

The cache is a uint8 tensor [pages, kv_heads, tiles, 34 * head_dim]: a tile holds 32 tokens of one head.  A value has
4 bits (sign, 2 exponent bits, 1 mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6), and 32 neighbouring values share a
power-of-two scale (a byte, exponent + 127; 255 stands for not a number).  A sequence's tokens are found through its
row of a page table.  What pages hold outside the written tokens is arbitrary bytes here, as in a program that
reuses pages.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TILE = 32
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # one decode step of 64 conversations puts its keys and values into the cache: latency
        {"name": "write step 64x8x128", "kind": "write", "batch": 64, "tokens": 64, "past": 2000, "kv": 8, "dim": 128,
         "page": 64, "dtype": "bf16", "fused": False},
        # three prompts of odd lengths, taken from a fused projection's fp32 output (strided rows)
        {"name": "write prompts 8190x8x128", "kind": "write", "batch": 3, "tokens": 8190, "past": 0, "kv": 8, "dim": 128,
         "page": 32, "dtype": "f32", "fused": True},
        # a prompt of the small model handed on as tensors
        {"name": "read 500x16x64", "kind": "read", "batch": 1, "tokens": 500, "start": 0, "kv": 16, "dim": 64,
         "page": 64, "dtype": "f32"},
        # the cache of 16 long conversations read back whole
        {"name": "read 65000x8x128", "kind": "read", "batch": 16, "tokens": 65000, "start": 21, "kv": 8, "dim": 128,
         "page": 128, "dtype": "bf16"},
        # one decode step of the small model after its 36-token prompt: the smallest call there is
        {"name": "cache 1x37 16/16x64", "kind": "cache", "batch": 1, "queries": 1, "length": 37, "spread": 1.0,
         "heads": 16, "kv": 16, "dim": 64, "page": 64, "dtype": "f32", "window": 0, "sinks": 0},
        # a decode step of 64 conversations of different lengths with shared heads
        {"name": "cache 64x8000 32/8x128", "kind": "cache", "batch": 64, "queries": 1, "length": 8000, "spread": 8.0,
         "heads": 32, "kv": 8, "dim": 128, "page": 64, "dtype": "bf16", "window": 0, "sinks": 0},
        # one very long document: few rows, a long axis
        {"name": "cache 1x131000 32/8x128", "kind": "cache", "batch": 1, "queries": 1, "length": 131000, "spread": 1.0,
         "heads": 32, "kv": 8, "dim": 128, "page": 128, "dtype": "f16", "window": 0, "sinks": 0},
        # many conversations that see their last 1024 tokens and the first 4
        {"name": "cache 128x16000 window 1024", "kind": "cache", "batch": 128, "queries": 1, "length": 16000,
         "spread": 4.0, "heads": 16, "kv": 4, "dim": 64, "page": 64, "dtype": "bf16", "window": 1024, "sinks": 4},
        # the next 512 tokens of a prompt over the 8190 before them
        {"name": "cache 512 over 8702 32/8x128", "kind": "cache", "batch": 1, "queries": 512, "length": 8702,
         "spread": 1.0, "heads": 32, "kv": 8, "dim": 128, "page": 64, "dtype": "bf16", "window": 0, "sinks": 0},
        # the small model's 36-token prompt: latency
        {"name": "prompt 36 16/16x64", "kind": "prompt", "batch": 1, "tokens": 36, "heads": 16, "kv": 16, "dim": 64,
         "dtype": "bf16", "window": 0, "sinks": 0},
        # eight prompts of different lengths packed one after another, all of the past visible
        {"name": "prompts 8x6001 16/16x64", "kind": "prompt", "batch": 8, "tokens": 6001, "heads": 16, "kv": 16,
         "dim": 64, "dtype": "f16", "window": 0, "sinks": 0},
        # a long prompt with shared heads and a window
        {"name": "prompt 8192 32/8x128 window", "kind": "prompt", "batch": 1, "tokens": 8192, "heads": 32, "kv": 8,
         "dim": 128, "dtype": "bf16", "window": 1024, "sinks": 4},
    ]


# ------------------------------------------------------------------ drawn cases

MOST_LOGITS = 2.2e9  # heads x rows x keys: what a plain form can hold in fp32, several times over


def _log_int(rng, low, high):
    return max(low, min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def _most(kind):
    """What the largest listed cases of a kind cost."""
    costs = [work(case) for case in listed() if case["kind"] == kind]
    return {key: max(cost[key] for cost in costs) for key in ("bytes", "flops")}


def draw(rng):
    kind = rng.choice(("write", "read", "cache", "cache", "cache", "prompt", "prompt"))
    most = _most(kind)
    while True:
        dim = rng.choice((64, 64, 128, 128, 128, 256))
        kv = rng.choice((1, 2, 3, 4, 8, 16))
        case = {"kind": kind, "kv": kv, "dim": dim, "dtype": rng.choice(("bf16", "f16", "f32"))}
        if kind in ("write", "read"):
            tokens = _log_int(rng, 1, 65000)
            case.update(batch=min(tokens, _log_int(rng, 1, 64)), tokens=tokens, page=rng.choice((32, 64, 128)))
            if kind == "write":
                case.update(past=rng.choice((0, _log_int(rng, 1, 4000))), fused=rng.random() < 0.5)
            else:
                case["start"] = rng.choice((0, _log_int(rng, 1, 1000)))
        else:
            case["heads"] = kv * rng.choice((1, 1, 2, 3, 4, 7, 8))
            case["window"] = rng.choice((0, 0, _log_int(rng, 1, 4096)))
            case["sinks"] = rng.choice((0, 1, 4, 40)) if case["window"] else 0
            if kind == "cache":
                length = _log_int(rng, 1, 131000)
                queries = min(length, rng.choice((1, 1, 1, 4, _log_int(rng, 2, 512))))
                case.update(batch=_log_int(rng, 1, 128), queries=queries, length=length,
                            spread=rng.choice((1.0, 2.0, 8.0)), page=rng.choice((32, 64, 128)))
            else:
                tokens = _log_int(rng, 1, 8192)
                case["dtype"] = rng.choice(("bf16", "f16"))
                case.update(tokens=tokens, batch=min(tokens, rng.choice((1, 1, 2, 8))))
        cost = work(case)
        if any(cost[key] > limit for key, limit in most.items()):
            continue
        if kind in ("cache", "prompt"):
            sizes = _sizes(case)
            keys = max(sizes["lengths"])
            if case["batch"] * case["heads"] * max(sizes["queries"]) * keys > MOST_LOGITS:
                continue
            if case["batch"] * case["kv"] * keys * dim > MOST_LOGITS / 2:
                continue
        return case


# ------------------------------------------------------------------ sizes


def _parts(total, batch, spread=3.0):
    """`total` in `batch` parts of at least one, the largest up to `spread` times the smallest, in no order."""
    weights = [1.0 + (spread - 1.0) * ((7 * i + 3) % batch) / max(1, batch - 1) for i in range(batch)]
    parts = [max(1, int(total * w / sum(weights))) for w in weights]
    index = 0
    while sum(parts) != total:
        step = 1 if sum(parts) < total else -1
        if parts[index % batch] + step >= 1:
            parts[index % batch] += step
        index += 1
    return parts


def _sizes(case):
    """New tokens (rows) and length of every sequence, in host numbers."""
    batch, kind = case["batch"], case["kind"]
    if kind == "cache":
        share = [1.0 if batch == 1 else 1.0 - (1.0 - 1.0 / case["spread"]) * ((5 * i + 2) % batch) / (batch - 1)
                 for i in range(batch)]
        lengths = [max(1, int(case["length"] * s)) for s in share]
        return {"queries": [min(case["queries"], n) for n in lengths], "lengths": lengths}
    rows = _parts(case["tokens"], batch)
    before = case.get("past", case.get("start", 0))
    return {"queries": rows, "lengths": [n + before for n in rows]}


def _visible(queries, length, window, sinks):
    """Visible (query, key) pairs of a sequence, and the keys that some query sees."""
    first = length - queries

    def seen(p):
        return p + 1 if window == 0 else min(p + 1, window) + min(sinks, max(0, p + 1 - window))

    pairs = sum(seen(p) for p in range(first, length))
    if window == 0:
        return pairs, length
    start = max(0, first - window + 1)
    return pairs, length - start + min(sinks, start)


def work(case):
    sizes = _sizes(case)
    rows, dim, kv = sum(sizes["queries"]), case["dim"], case["kv"]
    size = DTYPES[case["dtype"]].itemsize
    cached = dim * 17 // 32  # bytes of one head's row in the cache
    if case["kind"] == "write":  # in, into the cache and back out of it
        return {"bytes": 2 * rows * kv * (2 * dim * size + 2 * cached), "flops": 6 * rows * kv * dim}
    if case["kind"] == "read":
        return {"bytes": 2 * rows * kv * (dim * size + cached), "flops": 2 * rows * kv * dim}
    pairs, keys = map(sum, zip(*(_visible(q, n, case["window"], case["sinks"])
                                 for q, n in zip(sizes["queries"], sizes["lengths"]))))
    heads = case["heads"]
    values = 2 * keys * kv * cached if case["kind"] == "cache" else 2 * rows * kv * dim * size
    return {"bytes": values + 2 * rows * heads * dim * size, "flops": 4 * pairs * heads * dim}


# ------------------------------------------------------------------ inputs


def _generator(seed, part):
    return torch.Generator(device="cuda").manual_seed(1000003 * int(seed) + part)


def _offsets(counts):
    return torch.tensor([0] + counts, device="cuda").cumsum(0).to(torch.int32)


def _rows(generator, shape, spread=1.0):
    """N(0, spread) with 2% of the channels six times as large, as keys have them."""
    x = torch.randn(shape, generator=generator, device="cuda").mul_(spread)
    channels = torch.randperm(shape[-1], generator=generator, device="cuda")[:max(1, shape[-1] // 50)]
    x[..., channels] *= 6.0
    return x


def _pages(case, sizes, generator):
    """Empty pages and a page table: the sequences' pages lie scattered, table entries past them are -1."""
    page, kv, dim = case["page"], case["kv"], case["dim"]
    needed = [-(-n // page) for n in sizes["lengths"]]
    total = sum(needed) + 3
    shape = (total, kv, page // TILE, 34 * dim)
    pages = torch.randint(0, 256, shape, generator=generator, device="cuda", dtype=torch.uint8)
    order = torch.randperm(total, generator=generator, device="cuda").to(torch.int32)
    table = torch.full((len(needed), max(needed) + 2), -1, dtype=torch.int32, device="cuda")
    start = 0
    for row, count in enumerate(needed):
        table[row, :count] = order[start:start + count]
        start += count
    return pages, table


def prepare(case, seed):
    generator = _generator(seed, 1)
    kind, kv, dim, dtype = case["kind"], case["kv"], case["dim"], DTYPES[case["dtype"]]
    sizes = _sizes(case)
    rows = sum(sizes["queries"])
    state = {"kind": kind, "dtype": dtype, "rows": rows, "longest": max(sizes["lengths"]),
             "most": max(sizes["queries"]), "offsets": _offsets(sizes["queries"])}
    if kind == "prompt":
        state.update(window=case["window"], sinks=case["sinks"], **{
            name: _rows(generator, (rows, heads, dim)).to(dtype)
            for name, heads in (("q", case["heads"]), ("k", kv), ("v", kv))})
        return state
    pages, table = _pages(case, sizes, generator)
    state.update(pages=pages, table=table)
    lengths = torch.tensor(sizes["lengths"], dtype=torch.int32, device="cuda")
    if kind == "write":
        if case["fused"]:  # q, k and v side by side, as one projection leaves them
            fused = _rows(generator, (rows, 4 * kv, dim)).to(dtype)
            k, v = fused[:, 2 * kv:3 * kv], fused[:, 3 * kv:]
        else:
            k, v = (_rows(generator, (rows, kv, dim)).to(dtype) for _ in range(2))
        state.update(k=k, v=v, past=lengths - state["offsets"].diff())
        return state
    written = sizes["lengths"] if kind == "cache" else [n + case["start"] for n in sizes["queries"]]
    for row, length in enumerate(written):  # a sequence at a time, which bounds what is held at once
        k, v = (_rows(generator, (length, kv, dim)).to(torch.bfloat16) for _ in range(2))
        zero = torch.zeros(1, dtype=torch.int32, device="cuda")
        _write(pages, k, v, table[row:row + 1], zero, _offsets([length]))
    if kind == "read":
        state["start"] = lengths - state["offsets"].diff()
        return state
    state.update(q=_rows(generator, (rows, case["heads"], dim)).to(dtype), lengths=lengths, window=case["window"],
                 sinks=case["sinks"])
    return state


# ------------------------------------------------------------------ plain forms


def _places(pages, table, start, offsets, rows):
    """Of every row: its tile's number in pages.view(-1, bytes) for head 0, and its place in the tile."""
    row = torch.arange(rows, device="cuda")
    sequence = torch.searchsorted(offsets[1:].long(), row, right=True)
    position = start.long()[sequence] + row - offsets.long()[sequence]
    heads, tiles = pages.shape[1:3]
    page = table[sequence, position // (tiles * TILE)].long()
    return page * (heads * tiles) + position % (tiles * TILE) // TILE, position % TILE


def _addresses(pages, tile, place, dim):
    """Byte addresses in pages.view(-1) of the tokens' K codes, V codes, K scales and V scales, each
    [tokens, kv_heads, ...] with the head's bytes in the order of its dimensions."""
    heads, tiles, size = pages.shape[1:]
    width = dim // 32
    head = torch.arange(heads, device="cuda") * tiles
    base = ((tile[:, None] + head) * size)[..., None]
    t = place[:, None, None]
    byte = torch.arange(dim // 2, device="cuda")
    group = torch.arange(width, device="cuda")
    e, b = t // 16 * 4 + t % 4, t % 16 // 4
    per = 16 // width
    k = base + t * (dim // 2) + byte
    v = base + 16 * dim + e // per * 1024 + (b * 16 + byte // width) * 16 + e % per * width + byte % width
    return k, v, base + 32 * dim + group * 32 + t % 16 * 2 + t // 16, base + 33 * dim + group * 32 + b * 8 + e


def _quantise(x):
    """Codes (two to a byte) and scale bytes of [tokens, heads, dim]."""
    x = x.float()
    blocks = x.reshape(*x.shape[:-1], -1, 32)
    most = blocks.abs().amax(-1)
    bits = most.view(torch.int32)
    scale = ((bits + 0x200000) >> 23).sub(2).clamp(27, 252)
    inverse = torch.exp2((127 - scale).float())
    y = (blocks * inverse[..., None]).reshape(x.shape)
    a = y.abs()
    code = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = code + 8 * torch.signbit(y)
    code = code[..., 0::2] + 16 * code[..., 1::2]
    return code.to(torch.uint8), torch.where(most.isfinite(), scale, 255).to(torch.uint8)


def _values(codes, scales):
    """What codes [..., dim / 2] and scale bytes [..., dim / 32] stand for, in fp32."""
    table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device="cuda")
    nibbles = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    scale = torch.where(scales == 255, math.nan, torch.exp2(scales.float() - 127))
    return table[nibbles.int()] * scale.repeat_interleave(32, -1)


def _write(pages, k, v, table, past, offsets):
    tile, place = _places(pages, table, past, offsets, k.shape[0])
    at = _addresses(pages, tile, place, k.shape[-1])
    (k_codes, k_scales), (v_codes, v_scales) = _quantise(k), _quantise(v)
    flat = pages.view(-1)
    flat[at[0]], flat[at[1]], flat[at[2]], flat[at[3]] = k_codes, v_codes, k_scales, v_scales


def _read(pages, table, start, offsets, rows, dtype):
    tile, place = _places(pages, table, start, offsets, rows)
    at = _addresses(pages, tile, place, pages.shape[-1] // 34)
    flat = pages.view(-1)
    return (_values(flat[at[0]], flat[at[2]]).to(dtype), _values(flat[at[1]], flat[at[3]]).to(dtype))


def _softmax_product(q, k, v, seen, scale):
    """q [B, kv, group, n, D], k and v [B, kv, L, D], seen [B, n, L]: attention in fp32 with masked rows 0."""
    batch, kv, group, n, dim = q.shape
    scores = torch.matmul(q.reshape(batch, kv, group * n, dim), k.transpose(-1, -2)).mul_(scale)
    scores = scores.view(batch, kv, group, n, -1).masked_fill_(~seen[:, None, None], -math.inf)
    most = scores.amax(-1, keepdim=True).clamp_min_(-3e38)
    weights = scores.sub_(most).exp_()
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.view(batch, kv, group * n, -1), v).view(batch, kv, group, n, dim)
    return out / total.clamp_min(1e-38)


def _seen(positions, keys, window, sinks):
    key = torch.arange(keys, device="cuda")
    p = positions[..., None]
    seen = key <= p
    if window:
        seen = seen & ((key > p - window) | (key < sinks))
    return seen


def _pad(offsets, most):
    """Rows of every sequence, [B, most], and which of them it has."""
    starts, counts = offsets[:-1].long(), offsets.diff().long()
    index = torch.arange(most, device="cuda")
    return starts[:, None] + torch.minimum(index, (counts - 1).clamp_min(0)[:, None]), index < counts[:, None]


def _attend_cache(s):
    q, pages, table, lengths, dtype = s["q"], s["pages"], s["table"], s["lengths"].long(), s["dtype"]
    heads, tiles, size = pages.shape[1:]
    dim, longest = size // 34, s["longest"]
    batch = lengths.shape[0]
    key = torch.arange(longest, device="cuda").expand(batch, longest)
    page = table.gather(1, key // (tiles * TILE)).clamp_min(0).long()
    tile = page * (heads * tiles) + key % (tiles * TILE) // TILE
    at = _addresses(pages, tile.reshape(-1), (key % TILE).reshape(-1), dim)
    flat = pages.view(-1)
    there = (key < lengths[:, None])[:, None, :, None]
    k, v = (torch.where(there, _values(flat[a], flat[b]).view(batch, longest, heads, dim).transpose(1, 2), 0.0)
            for a, b in ((at[0], at[2]), (at[1], at[3])))
    row, has = _pad(s["offsets"], s["most"])
    positions = (lengths - s["offsets"].diff())[:, None] + torch.arange(s["most"], device="cuda")
    seen = _seen(positions, longest, s["window"], s["sinks"])
    grouped = q[row].float().view(batch, s["most"], heads, -1, dim).permute(0, 2, 3, 1, 4)
    out = _softmax_product(grouped, k, v, seen, dim ** -0.5).permute(0, 3, 1, 2, 4).reshape(batch, s["most"], -1, dim)
    result = torch.empty_like(q)
    result[row[has]] = out[has].to(dtype)
    return result


def _attend_prompt(s):
    q, k, v = s["q"], s["k"], s["v"]
    most, kv, dim = s["most"], k.shape[1], q.shape[-1]
    row, has = _pad(s["offsets"], most)
    batch = row.shape[0]
    grouped = q[row].float().view(batch, most, kv, -1, dim).permute(0, 2, 3, 1, 4)
    keys, values = (x[row].float().transpose(1, 2) for x in (k, v))
    positions = torch.arange(most, device="cuda").expand(batch, most)
    seen = _seen(positions, most, s["window"], s["sinks"])
    out = _softmax_product(grouped, keys, values, seen, dim ** -0.5)
    result = torch.empty_like(q)
    result[row[has]] = out.permute(0, 3, 1, 2, 4).reshape(batch, most, -1, dim)[has].to(s["dtype"])
    return result


def run(state):
    s = state
    if own:
        return _run_own(s)
    if s["kind"] == "write":
        _write(s["pages"], s["k"], s["v"], s["table"], s["past"], s["offsets"])
        return _read(s["pages"], s["table"], s["past"], s["offsets"], s["rows"], s["dtype"])
    if s["kind"] == "read":
        return _read(s["pages"], s["table"], s["start"], s["offsets"], s["rows"], s["dtype"])
    return _attend_cache(s) if s["kind"] == "cache" else _attend_prompt(s)


def _run_own(s):
    attention = s.get("module")
    if attention is None:
        package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ivonar-inference_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        from ivonar_amd import attention

        s["module"] = attention
    if s["kind"] == "write":
        attention.cache_write(s["pages"], s["k"], s["v"], s["table"], s["past"], s["offsets"])
        return attention.cache_read(s["pages"], s["table"], s["past"], s["offsets"], s["rows"], s["dtype"])
    if s["kind"] == "read":
        return attention.cache_read(s["pages"], s["table"], s["start"], s["offsets"], s["rows"], s["dtype"])
    if s["kind"] == "cache":
        return attention.cache_attention(s["q"], s["pages"], s["table"], s["lengths"], s["offsets"], s["window"],
                                         s["sinks"], max_length=s["longest"])
    return attention.window_attention(s["q"], s["k"], s["v"], s["offsets"], s["window"], s["sinks"])


# ------------------------------------------------------------------ answers in 64 bits


def _nearest(x):
    """The 4-bit value nearest to every x, ties to the even code, from the distances to all of them."""
    grid = torch.tensor(MAGNITUDES, dtype=torch.float64, device=x.device)
    out = torch.empty_like(x)
    for part, to in zip(x.flatten().split(1 << 22), out.view(-1).split(1 << 22)):
        distance = (part.abs()[:, None] - grid).abs()
        distance[:, 1::2] += (distance[:, 1::2] == distance.amin(1, keepdim=True)) * 1e-9  # odd codes lose ties
        to.copy_(torch.copysign(grid[distance.argmin(1)], part))
    return out


def _stored(x):
    """What the cache gives back for x [tokens, heads, dim] of finite values."""
    blocks = x.double().unflatten(-1, (-1, 32))
    most = blocks.abs().amax(-1, keepdim=True)
    exponent = torch.frexp(most * 8 / 7).exponent - 1 - 2
    exponent = torch.where(most > 0, exponent, -100).clamp(-100, 125).double()
    return (_nearest(blocks / 2.0 ** exponent) * 2.0 ** exponent).flatten(-2)


def _tile_values(tiles, dim):
    """K and V [heads, 32, dim] in 64 bits of tiles uint8 [heads, 34 * dim], one byte position at a time."""
    def four(code):
        low = code & 7
        value = torch.where(low < 2, low * 0.5, (1 + (low & 1) * 0.5) * 2.0 ** ((low >> 1) - 1))
        return torch.where(code >= 8, -value, value)

    def two(byte):
        return torch.stack((four(byte & 15), four(byte >> 4)), -1).double()

    tiles = tiles.long()
    heads, width = tiles.shape[0], dim // 32
    k = two(tiles[:, :16 * dim]).reshape(heads, 32, dim)
    v = two(tiles[:, 16 * dim:32 * dim]).reshape(heads, width // 2, 4, 16, 16 // width, 2 * width)
    v = v.permute(0, 1, 4, 2, 3, 5).reshape(heads, 2, 4, 4, dim).transpose(2, 3).reshape(heads, 32, dim)
    k_scale = tiles[:, 32 * dim:33 * dim].reshape(heads, width, 16, 2).permute(0, 3, 2, 1).reshape(heads, 32, width)
    v_scale = tiles[:, 33 * dim:].reshape(heads, width, 4, 2, 4).permute(0, 3, 2, 4, 1).reshape(heads, 32, width)
    return tuple((x.unflatten(-1, (-1, 32)) * 2.0 ** (e - 127).double()[..., None]).flatten(-2)
                 for x, e in ((k, k_scale), (v, v_scale)))


def _cached(pages, entries, length):
    """K and V [heads, length, dim] in 64 bits of the sequence whose pages are `entries`."""
    count, heads, tiles, size = pages.shape
    needed = -(-length // TILE)
    chosen = pages[entries[:-(-needed // tiles)].long()].transpose(0, 1).reshape(heads, -1, size)[:, :needed]
    k, v = _tile_values(chosen.reshape(-1, size), size // 34)
    return tuple(x.reshape(heads, -1, size // 34)[:, :length] for x in (k, v))


def _attention_64(q, k, v, first, window, sinks):
    """q [n, heads, dim] at positions first.., k and v [kv, length, dim], all in 64 bits."""
    n, heads, dim = q.shape
    out = torch.zeros_like(q)
    group = heads // k.shape[0]
    key = torch.arange(k.shape[1], device=q.device)
    for start in range(0, n, 1024):
        position = torch.arange(first + start, first + min(n, start + 1024), device=q.device)[:, None]
        hidden = key > position
        if window:
            hidden |= (key <= position - window) & (key >= sinks)
        for head in range(heads):
            scores = q[start:start + 1024, head] @ k[head // group].T / math.sqrt(dim)
            scores[hidden] = -math.inf
            out[start:start + 1024, head] = torch.softmax(scores, -1) @ v[head // group]
    return out


def exact(case, seed):
    state = prepare(case, seed)
    sizes, kind = _sizes(case), case["kind"]
    if kind == "write":
        return _stored(state["k"]), _stored(state["v"])
    results, start = [], 0
    for row, (count, length) in enumerate(zip(sizes["queries"], sizes["lengths"])):
        part = slice(start, start + count)
        start += count
        if kind == "prompt":
            k, v = (state[name][part].double().transpose(0, 1).contiguous() for name in ("k", "v"))
        else:
            k, v = _cached(state["pages"], state["table"][row], length)
        if kind == "read":
            results.append(tuple(x[:, length - count:].transpose(0, 1) for x in (k, v)))
        else:
            results.append(_attention_64(state["q"][part].double(), k, v, length - count, case["window"],
                                         case["sinks"]))
    if kind == "read":
        return torch.cat([k for k, _ in results]), torch.cat([v for _, v in results])
    return torch.cat(results)
